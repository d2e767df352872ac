"""Every form of the 8-bit product -- rows of a in LDS, shared out or streamed past; tiles of five sizes -- with each kind of scales and results, over
several blocks, a last one that ends early, last tiles that are partly empty, and rows that start anywhere."""
import math

import pytest

torch = pytest.importorskip("torch")

SCALES = [("e8m0", 1), ("e8m0", 128), ("f32", 1), ("f32", 128)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [(5, 400), (16, 17_000), (20, 5000), (257, 3001), (700, 6001), (300, 20_001), (1030, 13_000)]
LONG = [(16, 700, 8200)]                         # rows of a that take most of a compute unit's LDS
DIMS = [200, 385, 512]


def form(m, n, dim, exact, scale):
    """What a product of these sizes is made by: the rule of tv_fp8.hip, matmul()."""
    tiles = lambda tm, tn: -(-m // tm) * -(-n // tn)  # noqa: E731

    def time(tm, tn, held, rate):
        count, one = tiles(tm, tn), 256 * held
        return (-(-count // 256) if count <= one else -(-count // one) * held) * tm * tn / rate

    blocks = -(-dim // 128)
    if m <= 16 and dim >= 16:
        row = blocks * 128 + 16
        lds = m * row + blocks * 64 + 4096
        if m * row <= 64 << 10:
            return "shared out" if n < 256 * 4 * 16 else "streamed"
        if lds <= 160 << 10 and -(-n // 16) <= 256 * ((160 << 10) // lds):
            return "shared out"
    if exact and m <= 32:
        return 32, 128
    times = {(256, 256): math.inf if exact and scale == "f32" else time(256, 256, 1, 1.0), (128, 128): time(128, 128, 2, 0.88 if exact else 0.8),
             (64, 128): math.inf if tiles(64, 128) < 512 else time(64, 128, 3, 0.78 if exact else 0.72), (64, 64): time(64, 64, 4, 0.75 if exact else 0.58)}
    return min(times, key=times.get)


def test_sizes_reach_every_form():
    for exact in (True, False):
        for scale in ("e8m0", "f32"):
            for dim in DIMS:
                reached = {form(m, n, dim, exact, scale) for m, n in SIZES}
                every = {"shared out", "streamed", (64, 64), (64, 128), (128, 128)}
                every |= {(32, 128)} if exact else set()
                every |= set() if exact and scale == "f32" else {(256, 256)}
                assert reached == every, (exact, scale, dim)


def rows_of(fp8, rows, dim, scale, group, seed, odd):
    """8-bit rows as they are made, or at an odd place and stride with NaN codes between them."""
    x = torch.randn(rows, dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    x *= torch.exp2((torch.arange(rows, device="cuda") // 3 % 7 - 3).float())[:, None]
    r = fp8.quantize(x, scale=scale, group=group)
    if not odd:
        return r
    buffer = torch.full((rows * (dim + 3) + 64,), 0x7f, dtype=torch.uint8, device="cuda")
    codes = torch.as_strided(buffer, (rows, dim), (dim + 3, 1), 5)
    codes.copy_(r.codes.view(torch.uint8))
    return fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), r.scales, group)


def check(fp8, m, n, dim, scale, group):
    values = lambda r: r.codes.double() * r.scales.double().repeat_interleave(r.group, 0)[:len(r)].repeat_interleave(128, 1)[:, :dim]  # noqa: E731
    a, b = rows_of(fp8, m, dim, scale, 1, m + dim, False), rows_of(fp8, n, dim, scale, group, n + dim, False)
    x, y = values(a), values(b)
    want, size = x @ y.t(), (x * x) @ (y * y).t()
    for odd in (False, True):
        if odd:
            a, b = rows_of(fp8, m, dim, scale, 1, m + dim, True), rows_of(fp8, n, dim, scale, group, n + dim, True)
        for dtype in DTYPES:
            wide = torch.full((m + 1, n + 7), 3.0, dtype=dtype, device="cuda")
            out = wide[:m, 2:n + 2] if odd else torch.empty(m, n, dtype=dtype, device="cuda")
            fp8.matmul(a, b, out=out)
            # Of the root of the sum of squared products, which is what a result is about: 2^-24 for each of dim roundings, either way, and three a block for
            # the scales; into 16 bits up to seven products of eight cut off at 2^-13 of the largest, either way too, and half a step of the result.  Six
            # times that holds for millions of results; a result may be several times its usual size.
            step = torch.finfo(dtype).eps / 2
            usual = 2.0 ** -24 * (dim + 3 * -(-dim // 128)) ** 0.5 + (0 if dtype == torch.float32 else 2.0 ** -13 * 7 ** 0.5)
            off = (out.double() - want).abs()
            bound = 6 * usual * size.sqrt() + step * want.abs() * 1.001 + torch.finfo(dtype).smallest_normal * step
            over = want.abs() * (1 + step) >= torch.finfo(dtype).max
            assert bool(((off <= bound) | over).all()), (odd, dtype, float((off / bound)[~over].max()))
            if odd:
                wide[:m, 2:n + 2] = 3.0
                assert bool((wide == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale,group", SCALES)
@pytest.mark.parametrize("m,n", SIZES)
def test_forms(m, n, scale, group):
    from turbovec_amd import fp8
    for dim in DIMS:
        check(fp8, m, n, dim, scale, group)


@pytest.mark.gpu
@pytest.mark.parametrize("scale,group", SCALES)
@pytest.mark.parametrize("m,n,dim", LONG)
def test_forms_of_long_rows(m, n, dim, scale, group):
    from turbovec_amd import fp8
    assert form(m, n, dim, True, scale) == form(m, n, dim, False, scale) == "shared out"
    check(fp8, m, n, dim, scale, group)
