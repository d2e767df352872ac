"""Log probabilities, entropies and alternatives, and the scores' gradient, against the formulas in 64 bits.

Tolerances count roundings in 32 bits, u = 2^-24 each.  A slot's exponent (s - m) log2(e) / T is three roundings of itself, its exponential two u more; a
thread adds at most n / 64 + 64 terms one after the other, and a dozen more sums join threads and chunks.  So with D the mean of |d| = |s - m| / T under the softmax, log S is off by at most
(3 D + n / 64 + 80) u, log p by that and four roundings of its terms, the entropy log S + D by as much again and D's own: its terms p |d| are off by the same share, and as p's are."""
import math
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")
U = 2.0 ** -24


@pytest.fixture(scope="module")
def log_probs():
    from turbovec_amd import sampling
    return sampling.log_probs


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def words_of(allowed):
    """Mask words of truth values [..., n]."""
    n = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed, (0, -n % 64)).view(*allowed.shape[:-1], -1, 64)
    return (bits.long() << torch.arange(64, device="cuda")).sum(-1)


class Plain:
    """A row's distribution in 64 bits, and how far 32 bits may be off."""

    def __init__(self, scores, temperature=None, allowed=None):
        s = scores.detach().double()
        rows, n = s.shape
        t = torch.ones(rows, dtype=torch.float64, device="cuda") if temperature is None else temperature.double()
        if allowed is not None:
            s = torch.where(allowed, s, -INF)
        self.s, self.t, self.n = s, t, n
        self.empty = (s == -INF).all(1)
        top = torch.where(self.empty, 0.0, s.amax(1))
        d = (s - top[:, None]) / t[:, None]
        d[s == -INF] = -INF
        e = torch.exp(d)
        total = e.sum(1)
        self.d, self.log_sum = d, torch.where(self.empty, 0.0, total.log())
        self.log_p = torch.where(s == -INF, -INF, d - self.log_sum[:, None])
        self.p = torch.where(s == -INF, 0.0, e / total[:, None].clamp(min=1e-300))
        far = torch.where(s == -INF, 0.0, -d)
        self.mean, self.square = (self.p * far).sum(1), (self.p * far * far).sum(1)
        self.entropy = torch.where(self.empty, 0.0, self.log_sum + self.mean)
        self.off_sum = (3 * self.mean + n / 64 + 80) * U
        self.off_entropy = self.off_sum * (2 + self.mean) + 3 * self.square * U + 6 * (self.log_sum.abs() + self.mean) * U

    def off_log_p(self, log_p, d):
        return self.off_sum[:, None] + 4 * U * (d.abs() + self.log_sum.abs()[:, None])

    def at(self, slots):
        there = (slots >= 0) & (slots < self.n)
        i = slots.clamp(0, self.n - 1)
        lp, d = self.log_p.gather(1, i), self.d.gather(1, i)
        there &= lp > -INF
        return torch.where(there, lp, -INF), torch.where(there, d, 0.0), there

    def ranked(self, top):
        """Slots of the highest scores, ties to the lower one, and -1 behind the last."""
        order = torch.sort(self.s, dim=1, descending=True, stable=True).indices[:, :top]
        order = torch.where(self.s.gather(1, order) > -INF, order, -1)
        return torch.nn.functional.pad(order, (0, top - order.shape[1]), value=-1)

    def gradient(self, slots, g, g_entropy):
        """(gradient, what 32 bits may be off), unrounded."""
        lp, _, there = self.at(slots)
        g = torch.where(there, g.double(), 0.0)
        picked = torch.zeros_like(self.p).scatter_add_(1, slots.clamp(0, self.n - 1), g)
        picked_abs = torch.zeros_like(self.p).scatter_add_(1, slots.clamp(0, self.n - 1), g.abs())
        log_p = torch.where(self.p > 0, self.log_p, 0.0)
        towards = torch.where(self.p > 0, log_p + self.entropy[:, None], 0.0)
        ge = g_entropy.double()[:, None]
        want = (picked - self.p * (g.sum(1, keepdim=True) + ge * towards)) / self.t[:, None]
        far = torch.where(self.p > 0, -self.d, 0.0)
        off_l = self.off_sum[:, None] + 6 * U * (far + self.log_sum.abs()[:, None])            # of log p, which is what p is off by
        size = g.abs().sum(1, keepdim=True) + ge.abs() * (log_p.abs() + self.entropy[:, None])
        off = self.p * size * (off_l + 8 * U) + self.p * ge.abs() * (off_l + self.off_entropy[:, None]) + 130 * U * (picked_abs + self.p * g.abs().sum(1, keepdim=True))
        return want, off / self.t[:, None] + 4 * U * want.abs() + 2.0 ** -140


def check(log_probs, scores, slots, temperature=None, allowed=None, mask=None, top=0):
    """What a call finds against the plain form; `mask`, or the words of `allowed`."""
    if allowed is not None and mask is None:
        mask = words_of(allowed)
    found = log_probs(scores, slots, temperature=temperature, mask=mask, top=top)
    rows = len(scores)
    plain = Plain(scores, temperature if isinstance(temperature, torch.Tensor) else None if temperature is None else torch.full((rows,), temperature, device="cuda"), allowed)
    lp, d, there = plain.at(slots.view(rows, -1))
    got = found.log_probs.double().view(rows, -1)
    assert found.log_probs.shape == slots.shape and torch.equal(got == -INF, ~there)
    off = (got - lp).abs()[there] / plain.off_log_p(lp, d)[there]
    assert off.numel() == 0 or float(off.max()) <= 1, off.max()
    off = (found.entropy.double() - plain.entropy).abs() / plain.off_entropy
    assert float(off.max()) <= 1, off.max()
    assert found.top_slots.shape == found.top_log_probs.shape == (rows, top)
    if top:
        want = plain.ranked(top)
        assert torch.equal(found.top_slots, want)
        lp, d, there = plain.at(want)
        got = found.top_log_probs.double()
        assert torch.equal(got == -INF, ~there)
        off = (got - lp).abs()[there] / plain.off_log_p(lp, d)[there]
        assert off.numel() == 0 or float(off.max()) <= 1, off.max()
    return found


def check_gradient(log_probs, scores, slots, temperature=None, allowed=None, seed=1, mask=None):
    rows, n = scores.shape
    t = temperature if isinstance(temperature, torch.Tensor) else None if temperature is None else torch.full((rows,), temperature, device="cuda")
    g, ge = torch.randn(slots.shape, generator=gen(seed), device="cuda"), torch.randn(rows, generator=gen(seed + 1), device="cuda")
    scores = scores.detach().clone().requires_grad_(True)
    found = log_probs(scores, slots, temperature=temperature, mask=words_of(allowed) if allowed is not None and mask is None else mask)
    zero = torch.zeros_like(ge)
    plain = Plain(scores, t, allowed)
    for outputs, gradients in (((found.log_probs, found.entropy), (g, ge)), ((found.log_probs,), (g,)), ((found.entropy,), (ge,))):
        got, = torch.autograd.grad(outputs, scores, gradients, retain_graph=True)
        want, off = plain.gradient(slots.view(rows, -1), g.view(rows, -1) if found.log_probs is outputs[0] else torch.zeros_like(g).view(rows, -1), ge if outputs[-1] is found.entropy else zero)
        assert got.dtype == scores.dtype and got.shape == scores.shape
        half = torch.finfo(scores.dtype).eps / 2
        tolerance = off + half * (want.abs() + off) + (2.0 ** -25 if scores.dtype == torch.float16 else 0)
        assert bool(((got.double() - want).abs() <= tolerance).all()), ((got.double() - want).abs() / tolerance).max()
        if allowed is not None:
            assert bool((got[~allowed.expand(rows, n)] == 0).all())


def scores_of(rows, n, dtype, seed=1, spread=3.0):
    return (spread * torch.randn(rows, n, generator=gen(seed), device="cuda")).to(dtype)


def slots_of(rows, n, given, seed=2):
    return torch.randint(0, n, (rows, given), generator=gen(seed), device="cuda")


# ---- values ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 257, 1000, 2047, 2048, 2049, 4100, 10_007])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values(log_probs, n, dtype):
    for rows, given, top in ((1, 1, 1), (5, 3, 20), (40, 1, 0), (3, 128, 128)):
        check(log_probs, scores_of(rows, n, dtype), slots_of(rows, n, given), top=top)


@pytest.mark.parametrize("rows,n", [(1, 20_000), (1, 100_000), (3, 131_072), (300, 33_001), (1, 1_000_003), (7, 700_000), (2, 5_000_000), (1100, 9000)])
@pytest.mark.parametrize("dtype,top", [(torch.float32, 20), (torch.bfloat16, 5), (torch.float16, 128), (torch.bfloat16, 0)])
def test_long_rows(log_probs, rows, n, dtype, top):
    t = 0.5 + torch.rand(rows, generator=gen(3), device="cuda")
    check(log_probs, scores_of(rows, n, dtype, 4), slots_of(rows, n, 2), temperature=t, top=top)


@pytest.mark.parametrize("rows,n", [(4, 100), (3, 5000), (1, 300_000), (600, 2500)])
@pytest.mark.parametrize("share", [0.5, 0.01])
def test_masks(log_probs, rows, n, share):
    scores = scores_of(rows, n, torch.float32, 5)
    slots = slots_of(rows, n, 4)
    for shape in ((n,), (rows, n)):
        allowed = torch.rand(*shape, generator=gen(6), device="cuda") < share
        full = allowed.expand(rows, n)
        hidden = torch.where(full, scores, torch.tensor([float("nan"), INF, -INF, 3e38], device="cuda")[torch.arange(n, device="cuda") % 4])      # what is masked never counts
        check(log_probs, hidden, slots, allowed=full, mask=words_of(allowed), top=20)
        check_gradient(log_probs, hidden, slots, allowed=full, mask=words_of(allowed))


@pytest.mark.parametrize("n", [40, 3000, 200_000])
@pytest.mark.parametrize("rows", [6, 700])
def test_rows_that_allow_little_or_nothing(log_probs, rows, n):
    if rows * n > 30_000_000:
        rows = 20
    scores = scores_of(rows, n, torch.float32, 7)
    allowed = torch.rand(rows, n, generator=gen(8), device="cuda") < 0.5
    allowed[0] = False
    allowed[1] = False
    allowed[1, n - 1] = True
    scores[2] = -INF
    scores[3, :-2] = -INF
    allowed[3] = True
    scores[4] = torch.finfo(torch.float32).min                                   # the lowest value is a score
    slots = slots_of(rows, n, 3)
    slots[:, 0], slots[:2, 1] = n - 1, -1
    slots[3, 1] = n                                             # outside
    found = check(log_probs, scores, slots, allowed=allowed, top=7)
    assert found.top_slots[0].tolist() == [-1] * 7 and found.top_slots[1].tolist() == [n - 1] + [-1] * 6 and float(found.log_probs[1, 0]) == 0 and float(found.entropy[1]) == 0
    assert bool((found.top_log_probs[0] == -INF).all()) and float(found.entropy[0]) == 0 and float(found.entropy[2]) == 0
    check_gradient(log_probs, scores, slots, allowed=allowed)


@pytest.mark.parametrize("rows,n", [(3, 50), (3, 9000), (1, 300_000), (520, 3000)])
def test_nan_and_infinity(log_probs, rows, n):
    """They show in their row, and in no other."""
    rows = max(rows, 3)
    scores = scores_of(rows, n, torch.float32, 9)
    scores[0, n // 2], scores[2, 1] = float("nan"), INF
    slots = slots_of(rows, n, 2)
    slots[0, 1] = -1
    scores.requires_grad_(True)
    found = log_probs(scores, slots, top=4)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[0, 2]] = True
    assert torch.equal(torch.isnan(found.entropy), bad) and torch.equal(torch.isnan(found.log_probs[:, 0]), bad) and float(found.log_probs[0, 1]) == -INF
    order = torch.sort(torch.nan_to_num(scores.detach(), nan=-INF), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(found.top_slots, order)
    grad, = torch.autograd.grad(found.entropy.sum(), scores)
    assert torch.equal(torch.isnan(grad).any(1), bad)


@pytest.mark.parametrize("rows,n", [(2, 60), (2, 5000), (1, 400_000), (530, 2100)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_crowded_scores(log_probs, rows, n, dtype):
    """Ties: all equal; five values; the best ones a period apart, or all at one end, rising and falling."""
    slots = slots_of(rows, n, 1)
    ramp = torch.arange(n, device="cuda").float()
    for scores in (torch.zeros(rows, n), torch.randint(0, 5, (rows, n), generator=gen(10), device="cuda"), (ramp % 2048 == 5).expand(rows, n), (ramp % 64 < 8).expand(rows, n), (ramp / n * 20).expand(rows, n),
                   (-ramp / n * 20).expand(rows, n), (ramp > n - 200).expand(rows, n)):
        for top in (1, 20, 128):
            check(log_probs, scores.to("cuda").to(dtype).contiguous(), slots, top=top)


def test_temperatures(log_probs):
    """Of all sizes; at and below 0 the best slots share the mass, and there is no gradient."""
    scores = scores_of(9, 3000, torch.float32, 11)
    scores[6, 5], scores[6, 2000] = 50.0, 50.0
    t = torch.tensor([0.01, 100.0, 1e-6, 1e6, 3e-39, 1.0, 0.0, -2.0, float("nan")], device="cuda")
    slots = torch.stack((scores.argmax(1), scores.argmin(1)), 1)
    scores.requires_grad_(True)
    found = log_probs(scores, slots, temperature=t, top=3)
    check(log_probs, scores.detach()[:4], slots[:4], temperature=t[:4], top=3)
    assert found.log_probs[6].tolist()[1] == -INF and abs(float(found.log_probs[6, 0]) + math.log(2)) < 1e-6 and abs(float(found.entropy[6]) - math.log(2)) < 1e-6
    assert found.top_slots[6, :2].tolist() == [5, 2000] and float(found.top_log_probs[6, 2]) == -INF and int(found.top_slots[6, 2]) >= 0
    for row in (7, 8):
        assert found.log_probs[row].tolist() == [0.0, -INF] and float(found.entropy[row]) == 0
    assert found.log_probs[4].tolist() == [0.0, -INF]
    grad, = torch.autograd.grad(found.log_probs[:, 0].sum() + found.entropy.sum(), scores)
    assert bool((grad[6:] == 0).all()) and bool(torch.isfinite(grad).all())
    check(log_probs, scores.detach(), slots, temperature=0.3, top=3)


def test_large_scores(log_probs):
    """Differences that 32 bits do not hold, and scores far from 0."""
    scores = scores_of(4, 1000, torch.float32, 12)
    scores[0] += 1e5
    scores[1, ::2], scores[1, 1::2] = 3.0e38, -3.0e38
    scores[2] = torch.finfo(torch.float32).max
    scores[3, 7] = 1e30
    slots = slots_of(4, 1000, 3)
    found = log_probs(scores, slots, top=2)
    check(log_probs, scores[:1], slots[:1], top=2)
    assert abs(float(found.entropy[1]) - math.log(500)) < 1e-5 and abs(float(found.entropy[2]) - math.log(1000)) < 1e-5 and float(found.entropy[3]) == 0
    assert found.top_slots[1].tolist() == [0, 2] and found.top_slots[3, 0] == 7


@pytest.mark.parametrize("rows,n", [(5, 70), (5, 3001), (2, 100_001)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided(log_probs, rows, n, dtype):
    wide = scores_of(rows + 2, n + 9, dtype, 13)
    slots = torch.stack([slots_of(rows, n, 3)] * 2, 1)[:, 1]
    t = 0.5 + torch.rand(rows, generator=gen(14), device="cuda")
    for off in (0, 1, 3):
        scores = wide[1:-1, off:off + n]
        check(log_probs, scores, slots, temperature=t, top=9)
        check_gradient(log_probs, scores, slots, temperature=t)
    one = wide[:1, :n].expand(rows, n)                          # a row for all
    check(log_probs, one, slots, top=3)


# ---- gradients --------------------------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 64, 65, 1000, 2049, 8192, 10_007])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(log_probs, n, dtype):
    for rows, given in ((1, 1), (5, 3), (40, 1), (3, 128)):
        t = 0.5 + torch.rand(rows, generator=gen(15), device="cuda")
        check_gradient(log_probs, scores_of(rows, n, dtype, 16), slots_of(rows, n, given), temperature=t)


@pytest.mark.parametrize("rows,n", [(1, 100_000), (3, 131_073), (300, 33_001), (1, 2_000_003), (1100, 9000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_long_rows(log_probs, rows, n, dtype):
    check_gradient(log_probs, scores_of(rows, n, dtype, 17), slots_of(rows, n, 2))


@pytest.mark.parametrize("n", [3, 5000, 60_000])
def test_gradient_of_the_same_slot_twice(log_probs, n):
    slots = slots_of(4, n, 6)
    slots[:, 3] = slots[:, 0]
    slots[:, 5] = slots[:, 0]
    slots[1], slots[2, 1], slots[2, 2] = 2, -1, n + 5
    check_gradient(log_probs, scores_of(4, n, torch.float32, 18), slots)
    check_gradient(log_probs, scores_of(4, n, torch.bfloat16, 18), slots)


def test_gradient_against_differences(log_probs):
    """(f(s + h) - f(s - h)) / 2h, h = 2^-5: off by h^2 / 6 times the third derivative, below 2 / T^3 for both, and by the rounding of the two values, 2^-19 at most each here, over 2h."""
    rows, n, h = 3, 37, 2.0 ** -5
    scores, slots = scores_of(rows, n, torch.float32, 19, 1.0).requires_grad_(True), slots_of(rows, n, 1)
    for kind in (0, 1):
        f = lambda s: log_probs(s, slots, temperature=1.0)[kind].view(rows)      # noqa: E731
        grad, = torch.autograd.grad(f(scores).sum(), scores)
        for j in range(n):
            step = torch.zeros(n, device="cuda")
            step[j] = h
            with torch.no_grad():
                slope = (f(scores + step).double() - f(scores - step).double()) / (2 * h)
            assert float((slope - grad[:, j]).abs().max()) <= h * h / 3 + 2 * 2.0 ** -19 / (2 * h)


def test_gradient_through_a_loss(log_probs):
    """Sums and means spread one number over the rows; a second use of the scores adds up; no gradient, no graph."""
    scores, slots = scores_of(8, 500, torch.float32, 20).requires_grad_(True), slots_of(8, 500, 1)[:, 0]
    found = log_probs(scores, slots, temperature=0.8, top=3)
    assert found.log_probs.requires_grad and found.entropy.requires_grad and not found.top_log_probs.requires_grad
    loss = -found.log_probs.mean() - 0.01 * found.entropy.sum() + (scores * scores).sum() * 1e-3
    loss.backward()
    exact = scores.detach().double().requires_grad_(True)
    lp = torch.log_softmax(exact / 0.8, 1)
    (-lp.gather(1, slots[:, None]).mean() + 0.01 * (lp * lp.exp()).sum() + (exact * exact).sum() * 1e-3).backward()
    assert float((scores.grad.double() - exact.grad).abs().max()) <= 1e-6
    with torch.no_grad():
        assert not log_probs(scores, slots).log_probs.requires_grad
    assert not log_probs(scores.detach(), slots).log_probs.requires_grad
    found = log_probs(scores, slots)
    grad, = torch.autograd.grad(found.log_probs.sum(), scores, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), scores)


# ---- the rest -----------------------------------------------------------------------------------------

def test_same_bits_twice_and_beside_other_rows(log_probs):
    for rows, n in ((700, 3000), (5, 90_000)):
        scores, slots = scores_of(rows, n, torch.bfloat16, 21), slots_of(rows, n, 1)
        a, b = (log_probs(scores, slots, top=20) for _ in range(2))
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_no_rows_no_slots_many_rows(log_probs):
    scores = scores_of(5, 100, torch.float32, 22)
    found = log_probs(scores[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), top=4)
    assert found.log_probs.shape == (0,) and found.top_slots.shape == (0, 4)
    found = log_probs(scores, torch.zeros(5, 0, dtype=torch.int64, device="cuda"))
    assert found.log_probs.shape == (5, 0) and torch.isfinite(found.entropy).all()
    check_gradient(log_probs, scores_of(5, 100, torch.float32, 22), torch.zeros(5, 0, dtype=torch.int64, device="cuda"))
    rows = (1 << 22) + 5
    scores = torch.randn(rows, 3, generator=gen(23), device="cuda").half()
    slots = torch.arange(rows, device="cuda") % 3
    found = log_probs(scores.requires_grad_(True), slots, top=1)
    z = torch.log_softmax(scores.detach().double(), 1)
    assert float((found.log_probs.double() - z.gather(1, slots[:, None])[:, 0]).abs().max()) < 1e-5
    assert torch.equal(found.top_slots[:, 0], scores.argmax(1)) or bool((scores.detach().gather(1, found.top_slots) == scores.detach().amax(1, keepdim=True)).all())
    grad, = torch.autograd.grad(found.log_probs.sum(), scores)
    want = torch.nn.functional.one_hot(slots, 3) - z.exp()
    assert float((grad.double() - want).abs().max()) < 1e-3


def test_a_buffer_past_four_gigabytes(log_probs):
    rows, n = 300, 9000
    buffer = torch.empty(rows * 9_000_000, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(buffer, (rows, n), (9_000_000, 1), 0)
    far.copy_(scores_of(rows, n, torch.bfloat16, 24))
    check(log_probs, far, slots_of(rows, n, 2), top=5)
    check_gradient(log_probs, far, slots_of(rows, n, 2))


def test_refusals(log_probs):
    scores, slots = torch.zeros(4, 64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call, kind, text in (
            (lambda: log_probs(scores.t(), slots), ValueError, "contiguous"),
            (lambda: log_probs(scores[:, :0], slots), ValueError, "without scores"),
            (lambda: log_probs(scores, slots[:3]), ValueError, "slots must be of 4 rows"),
            (lambda: log_probs(scores, slots.int()), TypeError, "slots"),
            (lambda: log_probs(scores, slots.cpu()), ValueError, "slots must be on a GPU"),
            (lambda: log_probs(scores, torch.zeros(4, 129, dtype=torch.int64, device="cuda")), ValueError, "128"),
            (lambda: log_probs(scores, slots, top=129), ValueError, "top"),
            (lambda: log_probs(scores, slots, top=-1), ValueError, "top"),
            (lambda: log_probs(scores, slots, temperature=torch.ones(3, device="cuda")), ValueError, "temperature"),
            (lambda: log_probs(scores, slots, temperature=torch.ones(4, device="cuda").double()), TypeError, "temperature"),
            (lambda: log_probs(scores, slots, mask=torch.zeros(2, dtype=torch.int64, device="cuda")), ValueError, "mask"),
            (lambda: log_probs(scores, slots, mask=torch.zeros(1, device="cuda")), TypeError, "mask")):
        with pytest.raises(kind, match=text):
            call()


@pytest.mark.parametrize("rows,n", [(6, 4000), (1, 200_000)])
def test_on_another_stream_and_in_a_graph(log_probs, rows, n):
    scores, slots = scores_of(rows, n, torch.bfloat16, 25), slots_of(rows, n, 2)
    want = log_probs(scores, slots, top=10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = log_probs(scores, slots, top=10)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    leaf = scores.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = log_probs(scores, slots, top=10)
        found = log_probs(leaf, slots)
        grad, = torch.autograd.grad((found.log_probs.sum(), found.entropy.sum()), leaf)
    for seed in (26, 27, 28):
        scores.copy_(scores_of(rows, n, torch.bfloat16, seed))
        with torch.no_grad():
            leaf.copy_(scores)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, log_probs(scores, slots, top=10)))
        eager = scores.clone().requires_grad_(True)
        found = log_probs(eager, slots)
        want, = torch.autograd.grad((found.log_probs.sum(), found.entropy.sum()), eager)
        assert torch.equal(grad, want)


def test_two_threads(log_probs):
    scores, slots = scores_of(3, 150_000, torch.float32, 29), slots_of(3, 150_000, 2)
    want, wrong = log_probs(scores, slots, top=20), []
    torch.cuda.synchronize()

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = log_probs(scores, slots, top=20)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_a_draw_and_its_log_probability_agree(log_probs):
    """The same scores, temperature and mask to both: log p of what was drawn is the logarithm of its probability."""
    from turbovec_amd import sampling
    scores = scores_of(50, 20_000, torch.bfloat16, 30)
    allowed = torch.rand(50, 20_000, generator=gen(31), device="cuda") < 0.3
    allowed[7] = False
    mask, t = words_of(allowed), 0.5 + torch.rand(50, generator=gen(32), device="cuda")
    slots, p = sampling.sample(scores, torch.rand(50, generator=gen(33), device="cuda"), temperature=t, mask=mask)
    found = check(log_probs, scores, slots, temperature=t, allowed=allowed, top=1)
    assert int(slots[7]) == -1 and float(found.log_probs[7]) == -INF
    assert torch.allclose(found.log_probs.exp(), p, rtol=1e-4, atol=0)


# ---- rows with a workgroup each, a large one, two large ones to a compute unit, and rows in parts ---------------

FORMS = [(1, 8192), (1, 8193), (3, 20_001), (160, 16_400), (256, 9001), (257, 9001), (512, 8200), (513, 8200), (1, 100_600), (1, 100_601), (1, 8_388_608), (3, 2_800_007), (1, 9_000_001)]


@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("dtype,top", [(torch.float32, 24), (torch.bfloat16, 128), (torch.float16, 25), (torch.float32, 0)])
def test_forms(log_probs, rows, n, dtype, top):
    t = 0.5 + torch.rand(rows, generator=gen(40), device="cuda")
    scores, slots = scores_of(rows, n, dtype, 41), slots_of(rows, n, 3)
    scores[:, n - 1] = 40.0
    check(log_probs, scores, slots, temperature=t, top=top)
    allowed = torch.rand(rows, n, generator=gen(42), device="cuda") < 0.2
    allowed[rows // 2] = False
    check(log_probs, scores, slots, temperature=t, allowed=allowed, top=top)


@pytest.mark.parametrize("rows,n", [(1, 20_000), (200, 9000), (300, 9000), (1, 8_388_608), (2, 3_000_001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forms_of_crowded_scores(log_probs, rows, n, dtype):
    slots = slots_of(rows, n, 1)
    ramp = torch.arange(n, device="cuda").float()
    for scores in (torch.zeros(n), torch.randint(0, 5, (n,), generator=gen(43), device="cuda"), ramp % 2048 == 5, ramp % 64 < 8, ramp / n * 20, -ramp / n * 20, ramp > n - 200, (ramp > n // 3) & (ramp < n // 3 + 9000)):
        for top in (1, 128):
            check(log_probs, scores.to("cuda").to(dtype).expand(rows, n).contiguous(), slots, top=top)


@pytest.mark.parametrize("rows,n", [(4, 30_000), (200, 9000), (300, 9000), (4, 300_000)])
def test_forms_of_rows_that_show_or_have_nothing(log_probs, rows, n):
    scores = scores_of(rows, n, torch.float32, 44)
    scores[0, n // 2], scores[1, 1], scores[2] = float("nan"), INF, -INF
    slots = slots_of(rows, n, 2)
    found = log_probs(scores, slots, top=4)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[:2] = True
    assert torch.equal(torch.isnan(found.entropy), bad) and torch.equal(torch.isnan(found.log_probs).all(1), bad)
    assert bool((found.log_probs[2] == -INF).all()) and float(found.entropy[2]) == 0 and bool((found.top_slots[2] == -1).all())
    fine = log_probs(scores[3:], slots[3:], top=4)
    check(log_probs, scores[3:], slots[3:], top=4)
    assert all(torch.equal(x[3:], y) for x, y in zip(found, fine))          # (rows of the same form do not depend on what stands beside them)
    cold = log_probs(scores[3:], slots[3:], temperature=0.0, top=2)
    assert torch.equal(cold.top_slots, fine.top_slots[:, :2]) and bool((cold.log_probs[slots[3:] == cold.top_slots[:, :1]] == 0).all()) and bool((cold.entropy == 0).all())


def test_two_graphs_at_once(log_probs):
    """Rows in parts have a workspace: two captured calls, replayed on two streams at once, have one each."""
    scores, slots = [scores_of(2, 400_000, torch.float32, 45 + i) for i in range(2)], slots_of(2, 400_000, 2)
    want, graphs, got = [log_probs(s, slots, top=64) for s in scores], [], []
    for s in scores:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(log_probs(s, slots, top=64))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(50):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_what_a_call_may_also_be_given(log_probs):
    """Rows that are one and the same, slots out of a wider table, gradients of no rows; and a temperature that wants a gradient is refused."""
    one = scores_of(1, 3000, torch.float32, 50)
    table = slots_of(6, 3000, 5)
    t = torch.rand(6, generator=gen(51), device="cuda") + 0.5
    check(log_probs, one.expand(6, 3000), table[:, 1:4], temperature=t, top=3)
    check(log_probs, one.expand(6, 3000), table[:, 2].contiguous(), temperature=t)
    leaf = one.clone().requires_grad_(True)
    rows = leaf.expand(6, 3000)
    found = log_probs(rows, table[:, 1:4], temperature=t)
    got, = torch.autograd.grad((found.log_probs.sum(), found.entropy.sum()), leaf)
    plain = Plain(one.expand(6, 3000), t)
    want, off = plain.gradient(table[:, 1:4], torch.ones(6, 3, device="cuda"), torch.ones(6, device="cuda"))
    assert bool(((got.double() - want.sum(0)).abs() <= off.sum(0) + 2.0 ** -23 * want.abs().sum(0) * 6).all())
    none = torch.zeros(0, 100, device="cuda", requires_grad=True)
    found = log_probs(none, torch.zeros(0, 2, dtype=torch.int64, device="cuda"), top=2)
    grad, = torch.autograd.grad((found.log_probs.sum(), found.entropy.sum()), none)
    assert grad.shape == (0, 100)
    for scores in (one, leaf):
        with pytest.raises(ValueError, match="temperature has no gradient"):
            log_probs(scores, table[:1, 0], temperature=t[:1].clone().requires_grad_(True))
    with torch.no_grad():
        log_probs(one, table[:1, 0], temperature=t[:1].clone().requires_grad_(True))


@pytest.mark.parametrize("rows,n", [(1023, 700), (1024, 700), (1024, 1), (1500, 2048), (1500, 2049), (1100, 4096), (1100, 4097), (2000, 65), (1 << 16, 33)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_short_rows(log_probs, rows, n, dtype):
    """A wave to a row, and what is a little more than that."""
    t = 0.5 + torch.rand(rows, generator=gen(60), device="cuda")
    scores, slots = scores_of(rows, n, dtype, 61), slots_of(rows, n, 128)
    allowed = torch.rand(rows, n, generator=gen(62), device="cuda") < 0.5
    allowed[3] = False
    scores[5] = 1.0
    scores[6] = -INF
    scores[7, n // 2:] = 9.0
    for given, top in ((128, 24), (70, 25), (1, 1), (3, 0)):
        check(log_probs, scores, slots[:, :given], temperature=t, top=top)
        check(log_probs, scores, slots[:, :given], temperature=t, allowed=allowed, top=top)
    check_gradient(log_probs, scores, slots[:, :66], temperature=t)
    check_gradient(log_probs, scores, slots[:, :2], temperature=t, allowed=allowed)
    scores[8, n // 2], scores[9, 0] = float("nan"), INF
    found = log_probs(scores, slots, temperature=t, top=2)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[8:10] = True
    assert torch.equal(torch.isnan(found.entropy), bad) and torch.equal(torch.isnan(found.log_probs).all(1), bad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_short_rows_of_crowded_scores(log_probs, dtype):
    for n in (300, 2000):
        slots = slots_of(1024, n, 1)
        ramp = torch.arange(n, device="cuda").float()
        for scores in (torch.zeros(n), torch.randint(0, 5, (n,), generator=gen(63), device="cuda"), ramp % 512 == 5, ramp % 64 < 8, ramp / n * 20, -ramp / n * 20, ramp > n - 200):
            for top in (1, 24):
                check(log_probs, scores.to("cuda").to(dtype).expand(1024, n).contiguous(), slots, top=top)
