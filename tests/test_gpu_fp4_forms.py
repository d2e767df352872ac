"""Every form of the 4-bit product -- rows of b streamed past those of a, 16 of them to a wave or shared out over four or eight; tiles of five sizes, a last round's columns in
smaller ones, small tiles whose waves share the stages; rows too short or too far apart for those -- into each type, over rows that start anywhere, last tiles that are partly empty and last blocks that
are odd."""
import pytest

torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TILES = {(256, 256): (1, 1.44, 4.3, 1.4), (128, 128): (2, 0.59, 0.34, 0.42), (64, 64): (4, 0.23, 0.24, 0.14), (64, 128): (3, 0.39, 0.18, 0.3), (32, 128): (3, 0.27, 0.33, 0.19)}
SIZES = [(5, 400), (7, 9000), (16, 17_001), (17, 5000), (20, 70_003), (257, 3001), (700, 6001), (700, 6016), (1030, 13_007), (300, 40_001), (1030, 44_001)]
DIMS = [201, 385, 1500]
LONG = [(16, 700, 8199, "over eight"), (16, 9001, 8199, "tile"),          # rows of a that take most of a compute unit's LDS
        (17, 1000, 1793, "shared 32"), (40, 90, 2048, "shared 32"), (300, 700, 2049, "shared 32"), (33, 64, 2303, "shared 32"), (32, 1000, 2304, "shared 32"), (17, 31, 4100, "shared 32"),
        (64, 5001, 1281, "shared 64"), (64, 5001, 2048, "shared 64"), (130, 2500, 1537, "shared 64"), (70, 3333, 2303, "shared 64"), (128, 4000, 2305, "shared 64")]


def form(m, n, dim, size):
    """What a product of these sizes is made by: the rule of tv_fp4.hip, matmul4()."""
    def time(tile, n):
        tm, tn = tile
        held, stage, once, byte = TILES[tile]
        count, one = -(-m // tm) * -(-n // tn), 256 * held
        each = -(-count // 256) if count <= one else -(-count // one) * held
        return each * (-(-dim // 256) * stage + once + byte * size)

    def best(n):
        return min((t for t in TILES if t != (32, 128) or m <= 32), key=lambda t: time(t, n))

    if m <= 16 and dim >= 31:
        row, blocks = -(-dim // 128) * 64 + 16, -(-dim // 128)
        wide = -(-n // 16) <= 512
        lds = m * row + blocks * 64 + (8192 if wide else 4096)
        if m * row <= 64 << 10:
            return "streamed" if n >= 256 * 4 * 16 else "over eight" if wide else "over four"
        if lds <= 160 << 10 and -(-n // 16) <= 256 * ((160 << 10) // lds):
            return "over eight" if wide else "over four"
    if dim < 31:
        return "small"
    if dim > 7 * 256 and -(-m // 32) * -(-n // 32) <= 256:
        return "shared 32"
    if dim > 5 * 256 and -(-m // 64) * -(-n // 32) <= 256:
        return "shared 64"
    tile, mt, nt = best(n), -(-m // 256), -(-n // 256)
    if tile == (256, 256) and mt * nt > 256 and nt >= mt:
        columns = mt * nt // 256 * 256 // mt * 256
        if columns < n:
            rest = best(n - columns)
            if time(tile, columns) + time(rest, n - columns) + 3 < time(tile, n):
                return tile, rest
    return tile


def test_sizes_reach_every_form():
    reached = {form(m, n, dim, size) for m, n in SIZES for dim in DIMS for size in (2, 4)}
    assert {"over eight", "over four", "streamed", "shared 64", *TILES} <= reached, reached
    assert any(isinstance(f[0], tuple) for f in reached), reached
    for m, n, dim, what in LONG:
        assert (form(m, n, dim, 4) if what != "tile" else "tile" if form(m, n, dim, 4) in TILES else "") == what


def power(e):
    return torch.tensor([2.0 ** i for i in range(-200, 200)], dtype=torch.float64, device="cuda")[e.int() + 200]


def values64(r):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    grid = torch.cat((grid, -grid))
    c = torch.stack((r.codes & 15, r.codes >> 4), 2).view(len(r), -1)[:, :r.dim]
    return grid[c.int()] * power(r.scales.view(torch.uint8).int() - 127).repeat_interleave(32, 1)[:, :r.dim]


def rows_of(fp4, rows, dim, seed, stride=None):
    """4-bit rows as they are made, or at an odd place and stride with codes of -6 and scales that are NaN between them."""
    x = torch.randn(rows, dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    x *= torch.exp2((torch.arange(rows, device="cuda") // 3 % 7 - 3).float())[:, None]
    r = fp4.quantize(x)
    if stride is None:
        return r
    half, blocks = (dim + 1) // 2, -(-dim // 32)
    buffer = torch.full((rows * stride + 64,), 0xff, dtype=torch.uint8, device="cuda")
    codes = torch.as_strided(buffer, (rows, half), (stride, 1), 5)
    codes.copy_(r.codes)
    if dim % 2:
        codes[:, -1] |= 0xf0
    scales = torch.full((rows, blocks + 3), 255, dtype=torch.uint8, device="cuda")
    scales[:, 1:blocks + 1] = r.scales.view(torch.uint8)
    return fp4.Fp4Rows(codes, scales.view(torch.float8_e8m0fnu)[:, 1:blocks + 1], dim)


def check(fp4, m, n, dim, strides=None):
    """Each addition of a block's sum, which is exact, is off by 2^-23 at most of the sum of all magnitudes, the result by a rounding more."""
    a, b = rows_of(fp4, m, dim, m + dim), rows_of(fp4, n, dim, n + dim)
    x, y = values64(a), values64(b)
    want, most = x @ y.t(), x.abs() @ y.abs().t()
    most *= (-(-dim // 32) + 1) * 2.0 ** -23
    for odd in (False, True):
        if odd:
            a, b = (rows_of(fp4, r, dim, r + dim, s) for r, s in zip((m, n), strides or ((dim + 1) // 2 + 3,) * 2))
        for dtype in DTYPES:
            wide = torch.full((m + 1, n + 7), 3.0, dtype=dtype, device="cuda")
            out = wide[:m, 2:n + 2] if odd else torch.empty(m, n, dtype=dtype, device="cuda")
            fp4.matmul(a, b, out=out)
            tolerance = most + torch.finfo(dtype).eps / 2 * 1.001 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            over = want.abs() + tolerance >= torch.finfo(dtype).max
            off = (out.double() - want).abs()
            assert bool(((off <= tolerance) | over).all()), (odd, dtype, float((off / tolerance)[~over].max()))
            if odd:
                wide[:m, 2:n + 2] = 3.0
                assert bool((wide == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("m,n", SIZES)
def test_forms(m, n, dim):
    from turbovec_amd import fp4
    check(fp4, m, n, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,dim", [c[:3] for c in LONG] + [(1, 33, 30), (70, 1000, 17), (300, 2000, 30)])
def test_forms_of_long_and_short_rows(m, n, dim):
    from turbovec_amd import fp4
    check(fp4, m, n, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,dim", [(17, 130, 201), (40, 50, 1500)])
def test_rows_eight_megabytes_apart(m, n, dim):
    """A tile's offsets have 32 bits: rows a little nearer than 8 MB go through tiles, others do not, and either side may be the far one."""
    from turbovec_amd import fp4
    for far in ((1 << 23) - 1, 1 << 23, (1 << 23) + 5):
        check(fp4, m, n, dim, (far, (dim + 1) // 2))
        check(fp4, m, n, dim, ((dim + 1) // 2, far))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,dim,what", [(17, 150, 2100, "shared 32"), (64, 4200, 1600, "shared 64"), (9, 5000, 4097, "over eight"), (12, 9000, 1000, "over four")])
def test_nan_stays_in_its_row(m, n, dim, what):
    """Whichever waves have the block that it stands in, and wherever a row ends."""
    from turbovec_amd import fp4
    assert form(m, n, dim, 4) == what
    x, y = (torch.randn(r, dim, generator=torch.Generator(device="cuda").manual_seed(r), device="cuda") for r in (m, n))
    x[1, dim - 1], x[3, 300], y[5, 40], y[n - 1, 0], y[20, dim - 1] = float("nan"), float("inf"), float("inf"), float("nan"), float("inf")
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[[1, 3]], want[:, [5, 20, n - 1]] = True, True
    assert torch.equal(torch.isnan(fp4.matmul(fp4.quantize(x), fp4.quantize(y))), want)
