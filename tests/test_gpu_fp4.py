"""4-bit rows -- made, read back, multiplied -- against plain 64-bit forms of the same definitions, at the sizes, strides and values where
a byte, a block, a tile or a load ends."""
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@pytest.fixture(scope="module")
def fp4():
    from turbovec_amd import fp4
    return fp4


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def wild(rows, dim, seed, orders=20):
    """Values whose magnitudes differ by orders from row to row and within."""
    g = gen(seed)
    x = torch.randn(rows, dim, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, dim, generator=g, device="cuda"))
    return x * torch.exp2(torch.randint(-orders, orders, (rows, 1), generator=g, device="cuda").float())


def power(e):
    """2^e in 64 bits, exactly (the device's own powers are off by a rounding)."""
    return torch.tensor([2.0 ** i for i in range(-200, 200)], dtype=torch.float64, device="cuda")[e.int() + 200]


def plain_rows(x):
    """(values, scale bytes) by the definition, in 64 bits."""
    rows, dim = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -dim % 32)).view(rows, -1, 32)
    fine = torch.isfinite(x).all(2)
    most = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2)
    m, e = torch.frexp(most)                                # most = m * 2^e, 7 = 0.875 * 2^3
    e = torch.where(most > 0, e - 3 + (m >= 0.875).int(), -126).clamp(min=-126)
    s = power(e)
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    q = (x.abs() / s[..., None]).clamp(max=6.0)
    above = torch.searchsorted(grid, q.contiguous()).clamp(max=7)
    below = (above - 1).clamp(min=0)
    to_above, to_below = grid[above] - q, q - grid[below]
    pick = torch.where((to_below < to_above) | ((to_below == to_above) & (below % 2 == 0)), below, above)
    v = torch.copysign(grid[pick], x) * s[..., None]
    v[~fine] = float("nan")
    return v.view(rows, -1)[:, :dim], torch.where(fine, e + 127, 255).to(torch.uint8)


def values64(r):
    """What rows stand for, from their bytes, in 64 bits."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device="cuda")
    c = torch.stack((r.codes & 15, r.codes >> 4), 2).view(len(r), -1)[:, :r.dim]
    b = r.scales.view(torch.uint8)
    s = torch.where(b == 255, float("nan"), power(b.int() - 127))
    return grid[c.int()] * s.repeat_interleave(32, 1)[:, :r.dim]


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e300), torch.nan_to_num(b, nan=1e300)) and torch.equal(torch.isnan(a), torch.isnan(b))


def check_rows(fp4, x):
    r = fp4.quantize(x)
    v, s = plain_rows(x)
    assert torch.equal(r.scales.view(torch.uint8), s)
    assert same(values64(r), v)
    if x.shape[1] % 2:
        assert bool((r.codes[:, -1] < 16).all())            # nothing in the half byte behind an odd row
    return r


# ---- quantize, values -----------------------------------------------------------------------------

@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 2), (3, 7), (5, 31), (4, 32), (4, 33), (7, 63), (3, 65), (130, 200), (257, 1000), (64, 1536), (2, 16384), (3, 16383), (1000, 40)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize(fp4, rows, dim, dtype):
    x = wild(rows, dim, 1)
    check_rows(fp4, (x / x.abs().max() * 1000).to(dtype))


def test_quantize_special_values(fp4):
    """Blocks of zeros, of denormals, of the largest values, with a NaN or an infinity; maxima at the border between two powers."""
    x = torch.randn(40, 100, generator=gen(2), device="cuda")
    x[0] = 0
    x[1, 5], x[1, 40], x[1, 99] = float("nan"), float("inf"), -float("inf")
    x[2] *= 1e-40
    x[3] = 3.4e38
    x[4, :32], x[4, 32:64] = 6.999999, 7.0
    x[4, 64:96], x[4, 96:] = 3.4999998, 3.5
    x[5] = 2.0 ** -149
    x[6] = -0.0
    x[7] = 2.0 ** -126 * 7
    x[8] = 2.0 ** -126 * 6.9999995
    x[9, :32] = torch.linspace(0, 2.0 ** -125, 32, device="cuda")
    x[10] = torch.finfo(torch.float32).min
    r = check_rows(fp4, x)
    b = r.scales.view(torch.uint8)
    assert b[1].tolist() == [255, 255, 127 - 1, 255] or bool((b[1, [0, 1, 3]] == 255).all()) and int(b[1, 2]) != 255
    assert bool((b[0] == 1).all()) and bool((values64(r)[0] == 0).all())


def test_quantize_ties_go_to_even(fp4):
    middles = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    for scale in (1.0, 2.0 ** -126, 2.0 ** 100):
        x = torch.tensor([6.0] + middles + [-v for v in middles], device="cuda")[None] * scale
        got = (values64(check_rows(fp4, x))[0] / scale).tolist()
        assert got[:8] == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0] and got[8:] == [-0.0, -1.0, -1.0, -2.0, -2.0, -4.0, -4.0]


def test_quantize_strided_and_beside_others(fp4):
    """Rows inside a wider buffer, starting off every alignment, into codes and scales inside wider ones: nothing else changes."""
    from turbovec_amd import _lib as T
    base = wild(140, 700, 3)
    for off, dim in ((0, 256), (1, 257), (3, 255), (2, 6), (5, 97)):
        x = base[:, off:off + dim]
        want = fp4.quantize(x.contiguous())
        got = fp4.quantize(x)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales.view(torch.uint8), want.scales.view(torch.uint8))
        half, blocks = (dim + 1) // 2, -(-dim // 32)
        codes, scales = torch.full((142, 301), 0x55, dtype=torch.uint8, device="cuda"), torch.full((142, blocks + 3), 0x55, dtype=torch.uint8, device="cuda")
        T.check(T.lib().tv_fp4_quantize_dev(0, torch.cuda.current_stream().cuda_stream, x.data_ptr(), T.F32, x.stride(0), 140, dim, codes[1:].data_ptr() + off, 301, scales[1:].data_ptr(), blocks + 3))
        assert torch.equal(codes[1:141, off:off + half], want.codes) and torch.equal(scales[1:141, :blocks], want.scales.view(torch.uint8))
        codes[1:141, off:off + half] = 0x55
        scales[1:141, :blocks] = 0x55
        assert bool((codes == 0x55).all()) and bool((scales == 0x55).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_every_code_and_scale(fp4, dtype):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")[None].repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None].repeat(1, 16).view(torch.float8_e8m0fnu)
    for dim in (512, 511):
        r = fp4.Fp4Rows(codes, scales, dim)
        got, want = r.values(dtype), values64(r).to(dtype)                # (rounded once: 64 bits hold every value)
        assert got.dtype == dtype and same(got.double(), want.double())


@pytest.mark.parametrize("rows,dim,offset,pad", [(1, 1, 0, 16), (9, 5, 3, 7), (70, 33, 1, 17), (33, 1000, 5, 512), (5, 16383, 0, 8192)])
def test_values_strided(fp4, rows, dim, offset, pad):
    g = gen(4)
    buffer = torch.randint(0, 256, (rows * pad + offset + 64,), generator=g, device="cuda").to(torch.uint8)
    codes = torch.as_strided(buffer, (rows, (dim + 1) // 2), (pad, 1), offset)
    blocks = -(-dim // 32)
    scales = torch.randint(100, 150, (rows, blocks + 2), generator=g, device="cuda").to(torch.uint8).view(torch.float8_e8m0fnu)[:, :blocks]
    r = fp4.Fp4Rows(codes, scales, dim)
    assert torch.equal(r.values().double(), values64(r))


# ---- matmul ---------------------------------------------------------------------------------------

def stored(fp4, x, pad=None, offset=0):
    """4-bit rows of x inside a buffer of 0xff: rows at a stride of `pad`, `offset` bytes in, scales beside NaN bytes; the half byte behind an odd row is 0xf."""
    r = fp4.quantize(x)
    if pad is None:
        return r
    rows, dim = x.shape
    half, blocks = (dim + 1) // 2, -(-dim // 32)
    buffer = torch.full((rows * pad + offset + 64,), 0xff, dtype=torch.uint8, device="cuda")
    codes = torch.as_strided(buffer, (rows, half), (pad, 1), offset)
    codes.copy_(r.codes)
    if dim % 2:
        codes[:, -1] |= 0xf0
    scales = torch.full((rows, blocks + 5), 255, dtype=torch.uint8, device="cuda")
    scales[:, :blocks] = r.scales.view(torch.uint8)
    return fp4.Fp4Rows(codes, scales.view(torch.float8_e8m0fnu)[:, :blocks], dim)


def check_product(fp4, a, b, dtype, out=None):
    """Blocks' sums are exact, and each addition of one, and of an instruction's four, is off by 2^-23 at most of what it adds to, which the sum of all magnitudes bounds; the result is
    rounded once more.  (float16 and bfloat16: half a step, or float16's smallest number.)"""
    got = fp4.matmul(a, b, dtype=dtype, out=out)
    x, y = values64(a), values64(b)
    want, most = x @ y.t(), x.abs() @ y.abs().t()
    half = torch.finfo(dtype).eps / 2
    tolerance = (-(-a.dim // 32) + 1) * 2.0 ** -23 * most + half * want.abs() * (1 + 2.0 ** -10) + (2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149)
    assert got.dtype == dtype and got.shape == want.shape
    assert bool(((got.double() - want).abs() <= tolerance).all()), ((got.double() - want).abs() / tolerance).max()
    return got


SIZES = [(1, 1), (1, 17), (2, 300), (5, 33), (15, 64), (16, 1000), (17, 130), (31, 257), (33, 100), (64, 64), (65, 129), (100, 1000), (128, 256), (129, 300), (257, 513)]


@pytest.mark.parametrize("dim", [1, 2, 3, 31, 32, 33, 64, 65, 127, 128, 129, 160, 255, 256, 257, 384, 1000, 1001, 1536])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul(fp4, dim, dtype):
    for m, n in ((1, 20), (16, 100), (17, 70), (70, 130), (130, 260)):
        check_product(fp4, fp4.quantize(wild(m, dim, 5, 3) * 0.1), fp4.quantize(wild(n, dim, 6, 3) * 0.01), dtype)


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_sizes(fp4, m, n, dtype):
    for dim in (96, 520):
        check_product(fp4, fp4.quantize(wild(m, dim, 7, 3) * 0.1), fp4.quantize(wild(n, dim, 8, 3) * 0.01), dtype)


@pytest.mark.parametrize("m,n,dim", [(1, 20_000, 768), (16, 70_001, 200), (7, 66_000, 1000), (37, 5000, 1000), (300, 3000, 384), (1024, 2000, 1536), (700, 900, 4096), (2000, 2100, 256), (3, 50, 16384), (16, 40, 16384),
                                     (9, 3000, 16383), (64, 64, 16384), (4100, 300, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matmul_larger(fp4, m, n, dim, dtype):
    check_product(fp4, fp4.quantize(wild(m, dim, 9, 2)), fp4.quantize(wild(n, dim, 10, 2)), dtype)


@pytest.mark.parametrize("dim,pad,offset", [(1, 1, 0), (31, 16, 3), (33, 17, 0), (63, 40, 1), (256, 128, 0), (256, 131, 7), (255, 128, 5), (257, 144, 16), (1001, 512, 0), (1001, 501, 0), (640, 336, 8)])
@pytest.mark.parametrize("m,n", [(3, 40), (16, 500), (70, 200), (300, 530)])
def test_matmul_strided(fp4, dim, pad, offset, m, n):
    """What lies behind a row -- codes of 6, scales that are NaN, the half byte behind an odd row -- is not part of it."""
    a, b = stored(fp4, wild(m, dim, 11, 3), pad, offset), stored(fp4, wild(n, dim, 12, 3), pad, offset)
    out = torch.full((m, n + 9), 7.0, device="cuda")
    check_product(fp4, a, b, torch.float32, out=out[:, 2:n + 2])
    assert bool((out[:, :2] == 7).all()) and bool((out[:, n + 2:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [4, 61])
def test_matmul_into_wider_rows(fp4, dtype, n):
    for m in (3, 80):
        out = torch.full((m + 2, n + 3), 5.0, dtype=dtype, device="cuda")
        check_product(fp4, fp4.quantize(wild(m, 100, 13, 2) * 0.1), fp4.quantize(wild(n, 100, 14, 2) * 0.01), dtype, out=out[1:-1, 1:n + 1])
        out[1:-1, 1:n + 1] = 5.0
        assert bool((out == 5).all())


@pytest.mark.parametrize("m", [2, 16, 40, 200])
def test_matmul_nan_stays_in_its_row(fp4, m):
    x, y = wild(m, 300, 15, 2), wild(150, 300, 16, 2)
    x[1, 299], y[5, 40], y[149, 0] = float("nan"), float("inf"), float("nan")
    got = fp4.matmul(fp4.quantize(x), fp4.quantize(y))
    want = torch.zeros(m, 150, dtype=torch.bool, device="cuda")
    want[1], want[:, 5], want[:, 149] = True, True, True
    assert torch.equal(torch.isnan(got), want)


@pytest.mark.parametrize("m", [1, 16, 64, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_every_scale_byte(fp4, m, dtype):
    """Each scale of b against a scale that brings the product back: exact, at both ends."""
    codes = torch.randint(0, 256, (256, 16), generator=gen(17), device="cuda").to(torch.uint8)
    b = fp4.Fp4Rows(codes, torch.arange(256, dtype=torch.uint8, device="cuda")[:, None].view(torch.float8_e8m0fnu))
    for e in (0, 127, 254):
        a = fp4.Fp4Rows(torch.randint(0, 256, (m, 16), generator=gen(18), device="cuda").to(torch.uint8), torch.full((m, 1), e, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))
        got = fp4.matmul(a, b, dtype=dtype)
        x, y = values64(a), torch.nan_to_num(values64(b))
        want = (x @ y.t())
        want[:, 255] = float("nan")
        fits = torch.isnan(want) | (want.abs() < 2.0 ** 127)
        w = want.float().to(dtype)                       # (32 bits hold what is below 2^127 and a multiple of 2^-149)
        tiny = want.abs() < 2.0 ** -126                  # (what is below them may be lost)
        assert bool((torch.isnan(got) == torch.isnan(w))[fits].all())
        assert bool(((got.double() - w.double()).abs()[fits & ~tiny & torch.isfinite(w)] == 0).all())
        assert bool((got.double().abs()[tiny] <= 2.0 ** -126).all())


def test_matmul_with_nothing(fp4):
    some, none = fp4.quantize(wild(3, 64, 19)), fp4.quantize(wild(0, 64, 20))
    assert len(none) == 0 and none.values().shape == (0, 64)
    assert fp4.matmul(some, none).shape == (3, 0) and fp4.matmul(none, some).shape == (0, 3)


def test_refusals(fp4):
    from turbovec_amd import fp8
    x = torch.zeros(4, 64, device="cuda")
    r = fp4.quantize(x)
    for call, kind, text in (
            (lambda: fp4.quantize(x.t()), ValueError, "contiguous"),
            (lambda: fp4.quantize(torch.zeros(2, 16385, device="cuda")), ValueError, "dim must be"),
            (lambda: fp4.quantize(torch.zeros(2, 0, device="cuda")), ValueError, "dim must be"),
            (lambda: fp4.Fp4Rows(r.codes, r.scales, 66), ValueError, "codes of dim 66"),
            (lambda: fp4.Fp4Rows(r.codes, r.scales, 62), ValueError, "codes of dim 62"),
            (lambda: fp4.Fp4Rows(r.codes, r.scales[:, :1]), ValueError, "scales of"),
            (lambda: fp4.Fp4Rows(r.codes, r.scales.view(torch.uint8)), TypeError, "scales"),
            (lambda: fp4.Fp4Rows(r.codes, r.scales.cpu()), ValueError, "GPU"),
            (lambda: r.values(torch.float64), TypeError, "dtype"),
            (lambda: fp4.matmul(r, fp8.quantize(x)), TypeError, "Fp4Rows"),
            (lambda: fp4.matmul(r, fp4.quantize(x[:, :63])), ValueError, "dim 64 of a"),
            (lambda: fp4.matmul(r, r, dtype=torch.int32), TypeError, "dtype"),
            (lambda: fp4.matmul(r, r, out=torch.zeros(4, 5, device="cuda")), ValueError, "out must be"),
            (lambda: fp4.matmul(r, r, out=torch.zeros(4, 4)), ValueError, "GPU"),
            (lambda: fp4.matmul(r, r, out=torch.zeros(4, 8, device="cuda")[:, ::2]), ValueError, "contiguous")):
        with pytest.raises(kind, match=text):
            call()
    assert fp4.Fp4Rows(r.codes, r.scales, 63).dim == 63


# ---- streams, graphs, threads, far addresses --------------------------------------------------------

def test_on_another_stream_and_in_a_graph(fp4):
    g = gen(21)
    x, y = torch.randn(200, 500, generator=g, device="cuda"), torch.randn(40, 500, generator=g, device="cuda")
    want = fp4.matmul(fp4.quantize(y), fp4.quantize(x)).clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a = fp4.matmul(fp4.quantize(y), fp4.quantize(x))
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(a, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = fp4.quantize(x)
        out, back = fp4.matmul(fp4.quantize(y), rows), rows.values(torch.bfloat16)
    for seed in (22, 23, 24):
        x.copy_(torch.randn(200, 500, generator=gen(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fp4.matmul(fp4.quantize(y), fp4.quantize(x))) and torch.equal(back, fp4.quantize(x).values(torch.bfloat16))


def test_two_threads(fp4):
    x, y = wild(300, 400, 25, 2), wild(500, 400, 26, 2)
    a, b = fp4.quantize(x), fp4.quantize(y)
    want, wrong = fp4.matmul(a, b).clone(), []
    torch.cuda.synchronize()

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = fp4.matmul(fp4.quantize(x), fp4.quantize(y))
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@pytest.mark.parametrize("m", [3, 70])
def test_a_buffer_past_four_gigabytes(fp4, m):
    """Rows 24 KB apart, 200000 of them: offsets of codes and of what is read back pass 32 bits."""
    n, dim = 200_000, 96
    small = fp4.quantize(wild(n, dim, 27, 2))
    buffer = torch.empty(n * 24_000, dtype=torch.uint8, device="cuda")
    codes = torch.as_strided(buffer, (n, 48), (24_000, 1), 0)
    codes.copy_(small.codes)
    far = fp4.Fp4Rows(codes, small.scales, dim)
    q = fp4.quantize(wild(m, dim, 28, 2))
    assert torch.equal(fp4.matmul(q, far), fp4.matmul(q, small))
    assert torch.equal(fp4.matmul(far, q), fp4.matmul(small, q))
    assert torch.equal(far.values()[-5:], small.values()[-5:])
    again = fp4.quantize(torch.as_strided(buffer.view(torch.float32), (n, dim), (6000, 1), 0)[-3:].contiguous())
    assert len(again) == 3


def test_more_rows_than_a_grid_has(fp4):
    """2^20 workgroups of 256 threads take 2^28 runs of eight: rows of one coordinate take four threads each."""
    n = (1 << 26) + 1000
    x = torch.randint(-6, 7, (n, 1), generator=gen(29), device="cuda", dtype=torch.int8).half()
    r = fp4.quantize(x)
    v = r.values(torch.float16)
    near = (v - x).abs()
    assert float(near[:1000].max()) <= 1 and float(near[-1000:].max()) <= 1 and float(near.max()) <= 1
    assert bool((v[-1000:] != 0)[x[-1000:] != 0].all())


def test_a_result_past_four_gigabytes(fp4):
    """Rows of one block, whose sums are exact in every form: the same wherever in the result they stand."""
    m, n = 70_001, 40_000
    a, b = fp4.quantize(wild(m, 32, 30, 2)), fp4.quantize(wild(n, 32, 31, 2))
    got = fp4.matmul(a, b, dtype=torch.bfloat16)
    for i in (0, 26_843, 53_687, m - 1):
        row = fp4.Fp4Rows(a.codes[i:i + 1], a.scales[i:i + 1])
        assert torch.equal(got[i:i + 1], fp4.matmul(row, b, dtype=torch.bfloat16))
