"""The sums behind log probabilities: nothing is left out of them, and their errors do not grow with the row's length.

Roundings of u = 2^-24.  A term is off by two of itself and by three of its exponent, 3 D u of S with D the mean distance from the best score.  What a thread loads at once, at most 32 scores, it adds
for itself: 31 additions.  Those sums are joined one after the other: k additions, and where a batch brings a new largest score a product, an exponential and a distance more, 5.  Then come at
most 6 + 16 additions of a workgroup and 4 + 6 + 4 of a row's parts, with two products, and two roundings of the logarithm's value."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_log_probs import DTYPES, INF, U, Plain, check_gradient, gen, log_probs, scores_of, slots_of, words_of  # noqa: E402, F401

JOINED = 2 + 31 + 22 + 14 + 2 + 2


def near(found, plain, slots, batches, rises):
    """log p and entropy within what `batches` of a thread, `rises` of them with a new largest score, may lose."""
    off = (3 * plain.mean + JOINED + batches + 5 * rises) * U
    lp, d, there = plain.at(slots)
    got = found.log_probs.double()
    assert torch.equal(got == -INF, ~there)
    over = (got - lp).abs()[there] / (off[:, None] + 4 * U * (d.abs() + plain.log_sum.abs()[:, None]))[there]
    assert over.numel() == 0 or float(over.max()) <= 1, over.max()
    over = (found.entropy.double() - plain.entropy).abs() / (off * (2 + plain.mean) + 3 * plain.square * U + 6 * (plain.log_sum.abs() + plain.mean) * U)
    assert float(over.max()) <= 1, over.max()


@pytest.mark.parametrize("rows,n", [(1024, 100_000), (1024, 1_000_000), (200, 1_000_000), (1, 10_000_000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_term_many_times(log_probs, rows, n, dtype):  # noqa: F811
    """A score of 0 in each thread's first load and one that is lower everywhere else: additions of the same term to a sum between two powers of two round the same way each time."""
    first = 256 * 4 if dtype == torch.float32 else 256 * 8
    slots = torch.tensor([[0, n - 1]], device="cuda").expand(rows, 2).contiguous()
    for low in (-6.5, -7.0, -7.5, -8.0, -8.5, -9.0, -9.5, -10.0):
        one = torch.full((1, n), low, dtype=dtype, device="cuda")
        one[0, :4 * first:first // 256] = 0
        plain = Plain(one)
        found = log_probs(one.expand(rows, n), slots)
        for x in found[:2]:
            assert bool((x == x[:1]).all())
        found = found._replace(log_probs=found.log_probs[:1], entropy=found.entropy[:1])
        # (workgroups of 256 with 4096 floats or 8192 other scores at once have the most batches)
        near(found, plain, slots[:1], n / (4 * first) + 16, 4)


# Of all forms that a call may take: a wave, 256 and 1024 threads to a row, two workgroups to a compute unit, parts; no thread has more than 16 batches.
FORMS = [(1, 1000), (1, 8192), (1, 8193), (3, 20_001), (160, 16_400), (256, 9001), (257, 9001), (512, 8200), (513, 8200), (700, 100_000), (1, 100_600), (1, 100_601), (3, 131_072), (2000, 333), (1500, 2047), (1100, 4097),
         (2000, 70_001), (1, 8_388_608), (3, 2_800_007), (1, 9_000_001)]


@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("dtype,spread", [(torch.float32, 3.0), (torch.bfloat16, 3.0), (torch.float16, 0.1), (torch.float32, 0.0)])
def test_no_share_is_lost(log_probs, rows, n, dtype, spread):  # noqa: F811
    """Without a score that outweighs the others: random ones, those that hardly differ, those that are all the same."""
    at_once = min(rows, 3 + 2_000_000 // n)                             # (rows are compared some at a time, and some of them are given again)
    scores = scores_of(at_once, n, dtype, 80, spread).repeat(-(-rows // at_once), 1)[:rows]
    slots = slots_of(at_once, n, 3).repeat(-(-rows // at_once), 1)[:rows]
    slots[:, 0] = n - 1
    found = log_probs(scores, slots)
    for x in found[:2]:
        assert torch.equal(x[:at_once].repeat(-(-rows // at_once), *[1] * (x.dim() - 1))[:rows], x)
    near(found._replace(log_probs=found.log_probs[:at_once], entropy=found.entropy[:at_once]), Plain(scores[:at_once]), slots[:at_once], 16, 16)


@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_slot_counts(log_probs, rows, n, dtype):  # noqa: F811
    """A few slots have all of the mass between them, 1 / k each: the last ones, the first, some in each part and in each thread's loads."""
    for seed in range(3):
        some = torch.randint(0, n, (1500,), generator=gen(90 + seed), device="cuda")
        spaced = torch.arange(0, n, max(n // 1300, 1), device="cuda")
        places = torch.unique(torch.cat((some, spaced + seed if n > 10_000 else spaced[:1], torch.tensor([0, n - 1, n - 2, n - 7, n // 2], device="cuda"))).clamp(0, n - 1))
        k = len(places)
        one = torch.full((1, n), -60.0, dtype=dtype, device="cuda")
        one[0, places] = 0
        slots = torch.stack((places[torch.randint(0, k, (rows,), generator=gen(93 + seed), device="cuda")], torch.full((rows,), n - 1, device="cuda")), 1)
        found = log_probs(one.expand(rows, n), slots)
        # (k ones: each of their sums is exact; the others are 2^-86 of one)
        assert float((found.log_probs.double() + math.log(k)).abs().max()) <= (2 + 2 * math.log(k)) * U
        assert float((found.entropy.double() - math.log(k)).abs().max()) <= (2 + 2 * math.log(k)) * U
        allowed = torch.zeros(n, dtype=torch.bool, device="cuda")
        allowed[places[::2]] = True
        found = log_probs(one.expand(rows, n), slots[:, 1].contiguous(), mask=words_of(allowed))
        left = int(allowed.sum())
        assert float((found.entropy.double() - math.log(left)).abs().max()) <= (2 + 2 * math.log(left)) * U


@pytest.mark.parametrize("rows,n", [(1, 1000), (2, 20_001), (200, 9001), (1, 300_001), (1100, 700), (1100, 5000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_gradient_sums_to_nothing(log_probs, rows, n, dtype):  # noqa: F811
    """What a row's scores gain together is 0: the softmax does not see a shift."""
    scores = scores_of(rows, n, dtype, 95).requires_grad_(True)
    slots = slots_of(rows, n, 2)
    found = log_probs(scores, slots)
    grad, = torch.autograd.grad((found.log_probs.sum(), found.entropy.sum()), scores)
    size = grad.double().abs().sum(1)
    half = torch.finfo(dtype).eps / 2
    # (roundings of the results, half a step each, and of p: with its row's S and entropy, each off by what the sums may be, and what 16-bit floats hold below their normal numbers)
    plain = Plain(scores.detach())
    off = (3 * plain.mean + JOINED + 16 + 80) * U * (2 + plain.mean + plain.log_sum)
    assert bool((grad.double().sum(1).abs() <= size * half + (2 + plain.entropy) * (off + 8 * U) * 4 + n * (2.0 ** -25 if dtype == torch.float16 else 0)).all())
    check_gradient(log_probs, scores, slots)


@pytest.mark.parametrize("rows,n,top", [(1, 80_600, 0), (1, 80_601, 0), (64, 118_400, 0), (64, 118_401, 0), (1, 101_100, 1), (1, 101_101, 1), (1, 110_600, 20), (1, 110_601, 20), (3, 165_800, 128), (3, 165_801, 128),
                                        (159, 175_400, 0), (159, 175_401, 0), (160, 175_401, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_in_one_and_in_parts(log_probs, rows, n, top, dtype):  # noqa: F811
    """Both sides of where a row's scores go to one workgroup or to several."""
    at_once = min(rows, 8)
    scores = scores_of(at_once, n, dtype, 97).repeat(-(-rows // at_once), 1)[:rows]
    slots = slots_of(at_once, n, 3).repeat(-(-rows // at_once), 1)[:rows]
    found = log_probs(scores, slots, top=top)
    plain = Plain(scores[:at_once])
    near(found._replace(log_probs=found.log_probs[:at_once], entropy=found.entropy[:at_once]), plain, slots[:at_once], 24, 24)
    if top:
        assert torch.equal(found.top_slots[:at_once], plain.ranked(top))
    for x in found[:2]:
        assert torch.equal(x[:at_once].repeat(-(-rows // at_once), *[1] * (x.dim() - 1))[:rows], x)
