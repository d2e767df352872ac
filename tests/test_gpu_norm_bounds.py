"""Norms at the bounds that their header states, and within the roundings that they have.

Of u = 2^-24: a sum x + residual is off by one, in h itself and in the mean's root; 16 squares of a thread are added in 32 bits, half of what they lose reaches the root, and what follows is added in 64 bits;
the mean as a float half a rounding, its root, the quotient and two products one each."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_norm import DTYPES, EPS, KINDS, inputs, norm, row_values  # noqa: E402, F401

OFF = (1 + 1 + 8 + 0.5 + 4) * 2.0 ** -24
# 16, 32 and 64 lanes to a row; one run or two, a few waves or many
DIMS = [100, 128, 200, 500, 513, 1000, 2048, 2056, 4096, 8192, 8200, 16384]


def check(rows, h, weight, to, scale, eps=EPS):
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * weight.double()
    block, top = (32, 7.0) if to == "fp4" else (128, 448.0)
    dim = y.shape[1]
    most = torch.nn.functional.pad(y.abs(), (0, -dim % block)).view(len(y), -1, block).amax(2)
    s = rows.scales.double()
    if scale == "f32":
        assert bool(((s - (most / top).clamp(min=2.0 ** -126)).abs() <= s * (OFF + 2.0 ** -24)).all())
    else:
        assert bool((most <= top * s * (1 + OFF)).all()) and bool(((most >= top / 2 * s * (1 - OFF)) | (s == 2.0 ** -126)).all())
    wide = s.repeat_interleave(block, 1)[:, :dim]
    q = (y / wide).abs()
    half = torch.where(q < 2, 0.25, torch.where(q < 4, 0.5, 1.0)) if to == "fp4" else torch.clamp(torch.exp2(torch.floor(torch.log2(q.clamp(min=2.0 ** -40)))) * 2.0 ** -4, min=2.0 ** -10)
    over = (row_values(rows) - y).abs() / wide - half - (2 * OFF + 2.0 ** -23) * q
    assert float(over.max()) <= 1e-9, over.max()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("to,scale", KINDS)
def test_roundings(norm, dim, dtype, to, scale):  # noqa: F811
    x, r, w = inputs(70, dim, dtype, 21)
    check(norm.rms_norm(x, w, eps=EPS, to=to, scale=scale), x.double(), w, to, scale)
    made, _ = norm.add_rms_norm(x, r, w, eps=EPS, to=to, scale=scale)
    check(made, x.double() + r.double(), w, to, scale)
    x[:] = 3.0                                          # (squares that round the same way each time)
    x[:, ::7] = 1.1
    check(norm.rms_norm(x, w, eps=EPS, to=to, scale=scale), x.double(), w, to, scale)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("to,scale", KINDS)
def test_the_largest_and_the_smallest_rows(norm, dim, dtype, to, scale):  # noqa: F811
    """Below 2^62 throughout a row has its norm, from 2^64 on it has none; at 2^-63 its squares are numbers, below 2^-75 eps is what remains."""
    one = torch.ones(dim, device="cuda")
    x = torch.full((3, dim), 2.0 ** 62 * (1 - torch.finfo(dtype).eps / 2), dtype=dtype, device="cuda")
    x[1, ::3] *= -0.5
    check(norm.rms_norm(x, eps=0, to=to, scale=scale), x.double(), one, to, scale, 0.0)
    if dtype == torch.float32:
        check(norm.add_rms_norm(x, -x * 2.0 ** -3, eps=0, to=to, scale=scale)[0], x.double() * 0.875, one, to, scale, 0.0)
    x[:, dim - 1] = 2.0 ** 64
    assert bool(torch.isnan(row_values(norm.rms_norm(x, to=to, scale=scale))).all())
    x[:] = 2.0 ** -63
    x[1, ::3] *= -4.0
    check(norm.rms_norm(x, eps=0, to=to, scale=scale), x.double(), one, to, scale, 0.0)
    x[:] = 2.0 ** -76
    check(norm.rms_norm(x, eps=2.0 ** -120, to=to, scale=scale), x.double(), one, to, scale, 2.0 ** -120)
    assert bool(torch.isnan(row_values(norm.rms_norm(x, eps=0, to=to, scale=scale))).all())
