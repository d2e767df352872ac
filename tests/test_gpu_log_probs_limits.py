"""Log probabilities where a parameter or a score is at its limit, in every form that a call may take."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_log_probs import DTYPES, INF, U, check, check_gradient, gen, log_probs, scores_of, slots_of  # noqa: E402, F401

# A wave to a row, workgroups of 256 and of 1024 threads, rows in parts; rows that end with a load of all types, and rows that do not.
FORMS = [(5, 1), (5, 7), (3, 1003), (3, 1008), (1030, 333), (1030, 1000), (1030, 2500), (2, 20_001), (200, 9003), (300, 9003), (2, 300_001), (2, 300_032)]


@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinite_temperature(log_probs, rows, n, dtype):  # noqa: F811
    """Slots that have a probability share the mass, whatever is masked, -infinity or behind the row's end; the gradient is 0.  (A sum of equal terms loses what its additions do: log S is off by no more than
    check allows, and a hundred roundings; the logarithm by two of itself.)"""
    scores, slots = scores_of(rows, n, dtype, 70), slots_of(rows, n, 2)
    t = torch.full((rows,), INF, device="cuda")
    scores[0, n // 2] = -INF
    slots[:, 0] = n // 2
    check(log_probs, scores, slots, temperature=t, top=3)
    check_gradient(log_probs, scores, slots, temperature=t)
    allowed = torch.rand(rows, n, generator=gen(71), device="cuda") < 0.5
    allowed[rows - 1] = False
    allowed[rows - 1, n - 1] = True
    allowed[1] = False
    found = check(log_probs, scores, slots, temperature=INF, allowed=allowed, top=3)
    there = (allowed & (scores > -INF)).sum(1).double()
    want = torch.where(there > 0, there.log(), 0.0)
    assert bool(((found.entropy.double() - want).abs() <= (100 + 2 * want) * U).all())
    check_gradient(log_probs, scores, slots, temperature=t, allowed=allowed)
    if rows > 2:                                       # beside rows of other temperatures
        t[1::2] = 0.7
        check(log_probs, scores, slots, temperature=t, allowed=allowed, top=3)
        check_gradient(log_probs, scores, slots, temperature=t, allowed=allowed)


def test_the_largest_temperatures(log_probs):  # noqa: F811
    """Scores as far apart as 32 bits hold, at temperatures whose inverse is no normal number; what lies further from the best has no probability."""
    low, high = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    scores = torch.tensor([[0.0, low / 2, low, -1.0, 0.0]] * 4, device="cuda")
    slots = torch.arange(5, device="cuda").expand(4, 5).contiguous()
    t = torch.tensor([high, 1e38, 2.0 ** 126, INF], device="cuda")
    check(log_probs, scores[:3], slots[:3], temperature=t[:3], top=5)
    found = log_probs(scores, slots, temperature=t)
    assert float((found.log_probs[3] + math.log(5)).abs().max()) <= 2.0 ** -20          # (the smallest factor times the largest distance is 2^-21)
    scores = torch.tensor([[high, low, high]], device="cuda")
    for temperature in (1.0, INF):
        found = log_probs(scores, slots[:1, :3].contiguous(), temperature=temperature, top=3)
        assert float(found.log_probs[0, 1]) == -INF and float((found.log_probs[0, ::2] + math.log(2)).abs().max()) < 1e-6 and abs(float(found.entropy[0]) - math.log(2)) < 1e-6
        assert found.top_slots.tolist() == [[0, 2, 1]]


@pytest.mark.parametrize("rows,n", FORMS)
def test_no_distance_is_too_small_for_the_limit(log_probs, rows, n):  # noqa: F811
    """At a temperature of 0 the best slots share the mass, however little the others lie below them."""
    if n < 7:
        return
    low = 2.0 ** -149
    for dtype, step in ((torch.float32, 3 * low), (torch.float32, 1e-39), (torch.bfloat16, 2.0 ** -133), (torch.float16, 2.0 ** -24)):
        scores = torch.zeros(rows, n, device="cuda", dtype=dtype)
        best = [1, n // 2, n - 1]
        scores[:, best] = step
        slots = torch.tensor([best + [0]], device="cuda").expand(rows, 4).contiguous()
        found = log_probs(scores, slots, temperature=0.0, top=4)
        assert float((found.log_probs[:, :3] + math.log(3)).abs().max()) <= 4 * U and bool((found.log_probs[:, 3] == -INF).all())
        assert float((found.entropy - math.log(3)).abs().max()) <= 4 * U
        assert bool((found.top_slots == torch.tensor(best + [0], device="cuda")).all()) and bool((found.top_log_probs[:, 3] == -INF).all())
        found = log_probs(-scores, slots, temperature=-1.0)                        # the best are all others
        assert float((found.log_probs[:, 3] + math.log(n - 3)).abs().max()) <= (100 + 2 * math.log(n)) * U and bool((found.log_probs[:, :3] == -INF).all())
    scores = torch.zeros(rows, n, device="cuda")
    scores[:, best] = 1e-40
    found = log_probs(scores, slots, temperature=1e-40)                            # no normal number
    assert float((found.log_probs[:, :3] + math.log(3)).abs().max()) <= 4 * U and bool((found.log_probs[:, 3] == -INF).all())


@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_signalling_nan_hides_no_score(log_probs, rows, n, dtype):  # noqa: F811
    """A NaN of any kind shows in the row's sums and is not among its best slots; those beside it are."""
    if n < 20:
        return
    bits, kind = {torch.float32: (0x7f800001, torch.int32), torch.float16: (0x7c01, torch.int16), torch.bfloat16: (0x7f81, torch.int16)}[dtype]
    scores = scores_of(rows, n, dtype, 72)
    for at in {0, 1, 6, n // 2, n - 2, n - 1}:
        scores[:, max(at - 1, 0):at + 2] = 20.0 + at / n
    order = scores.clone()
    for at in (1, n // 2, n - 1):
        scores.view(kind)[:, at] = bits
        order[:, at] = -INF
    found = log_probs(scores, slots_of(rows, n, 2), top=6)
    assert bool(torch.isnan(found.entropy).all()) and bool(torch.isnan(found.log_probs).all())
    assert torch.equal(found.top_slots, torch.sort(order, dim=1, descending=True, stable=True).indices[:, :6])
