"""8-bit rows -- made, multiplied, re-scored -- against plain 64-bit forms of the same definitions, at the sizes, strides and
values where a tile, a block or a load ends."""
import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def fp8():
    from turbovec_amd import fp8
    return fp8


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def wild(rows, dim, seed):
    """Values whose magnitudes differ by orders from block to block and within."""
    g = gen(seed)
    x = torch.randn(rows, dim, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, dim, generator=g, device="cuda"))
    return x * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g, device="cuda").float())


def spread(scales, group, rows, dim):
    return scales.double().repeat_interleave(group, 0)[:rows].repeat_interleave(128, 1)[:, :dim]


def values(r):
    return r.codes.double() * spread(r.scales, r.group, *r.codes.shape)


# ---- quantize -------------------------------------------------------------------------------------

def check_rows(fp8, x, scale, group):
    r = fp8.quantize(x, scale=scale, group=group)
    rows, dim = x.shape
    x = x.double()
    fine = torch.isfinite(x)
    padded = torch.nn.functional.pad(torch.where(fine, x.abs(), 0.0), (0, -dim % 128, 0, -rows % group))
    most = padded.view(-1, group, padded.shape[1] // 128, 128).amax((1, 3))
    if scale == "f32":
        # the rounded quotient: 53 bits are more than 2 * 24 + 2, so that rounding to them first changes nothing (a tensor
        # divided by a number would be multiplied by its reciprocal)
        want = torch.clamp((most / torch.full_like(most, 448.0)).float(), min=2.0 ** -126)
        assert torch.equal(r.scales, want)
    else:
        s = r.scales.double()
        assert r.scales.dtype == torch.float8_e8m0fnu
        assert bool((most <= 448 * s).all())                           # it fits
        assert bool(((most > 224 * s) | (s == 2.0 ** -126)).all())     # and would not with half of it
    q = x / spread(r.scales, group, rows, dim)
    c = r.codes.double()
    assert torch.equal(torch.isnan(c), ~fine)
    # the nearest code: half a step of 3 mantissa bits, 2^-10 below 2^-6; the quotient was rounded to 32 bits first
    half = torch.clamp(torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -40)))) * 2.0 ** -4, min=2.0 ** -10)
    off = torch.where(fine, (c - q).abs(), 0.0)
    assert bool((off <= torch.where(fine, half + q.abs() * 2.0 ** -23, 0.0)).all())
    return r


@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 127), (4, 128), (4, 129), (130, 200), (257, 1000), (64, 1536), (128, 128), (300, 385)])
@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("e8m0", 128), ("f32", 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize(fp8, rows, dim, scale, group, dtype):
    x = wild(rows, dim, 1)
    check_rows(fp8, (x / x.abs().max() * 1000).to(dtype), scale, group)


@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("group", [1, 128])
def test_quantize_special_values(fp8, scale, group):
    """Blocks of zeros, of nothing finite, of denormals, of the largest values; maxima at the border between two powers."""
    x = torch.randn(260, 512, generator=gen(2), device="cuda")
    x[0] = 0
    x[1, :128] = float("nan")
    x[1, 200] = float("inf")
    x[1, 201] = -float("inf")
    x[2] *= 1e-40
    x[3] = 3.4e38
    x[4, :128] = 448.0
    x[4, 128:256] = 448.00003
    x[4, 256:384] = 3.5
    x[4, 384:] = 2.0 ** -126 * 448
    x[5] = 2.0 ** -149
    x[6] = -0.0
    if group == 128:
        x = x.repeat_interleave(128, 0)[:128 * 7 + 3]
    r = check_rows(fp8, x, scale, group)
    assert bool((r.codes[0].float() == 0).all()) and bool((r.scales[0].double() == 2.0 ** -126).all())


def test_quantize_ties_go_to_even(fp8):
    x = torch.tensor([448.0] + [v for v in (1.0625, 1.1875, 1.3125, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10)] + [0.0] * 120, device="cuda")[None]
    c = fp8.quantize(x, scale="f32").codes.float()[0, 1:8].tolist()
    assert c == [1.0, 1.25, 1.25, 16.0, 20.0, 0.0, 2.0 ** -8]


@pytest.mark.parametrize("scale,group", itertools.product(["e8m0", "f32"], [1, 128]))
def test_quantize_strided_and_beside_others(fp8, scale, group):
    """Rows inside a wider buffer, starting off every alignment, into codes and scales inside wider ones: nothing else changes."""
    from turbovec_amd import _lib as T
    base = wild(140, 700, 3)
    for off, dim in ((0, 256), (1, 256), (3, 255), (128, 300)):
        x = base[:, off:off + dim]
        want = fp8.quantize(x.contiguous(), scale=scale, group=group)
        got = fp8.quantize(x, scale=scale, group=group)
        assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scales.view(torch.uint8), want.scales.view(torch.uint8))
        codes = torch.full((142, 512), 0x55, dtype=torch.uint8, device="cuda")
        blocks, size = -(-dim // 128), 1 if scale == "e8m0" else 4
        scales = torch.full((-(-140 // group) + 2, blocks + 3, size), 0x55, dtype=torch.uint8, device="cuda")
        T.check(T.lib().tv_fp8_quantize_dev(0, torch.cuda.current_stream().cuda_stream, x.data_ptr(), T.F32, x.stride(0), 140, dim, T.SCALE_E8M0 if scale == "e8m0" else T.SCALE_F32, group,
                                            codes[1:].data_ptr() + off, 512, scales[1:].data_ptr(), blocks + 3))
        assert torch.equal(codes[1:141, off:off + dim], want.codes.view(torch.uint8))
        assert torch.equal(scales[1:-1, :blocks].reshape(-(-140 // group), -1), want.scales.view(torch.uint8).reshape(-(-140 // group), -1))
        codes[1:141, off:off + dim] = 0x55
        scales[1:-1, :blocks] = 0x55
        assert bool((codes == 0x55).all()) and bool((scales == 0x55).all())


# ---- matmul ---------------------------------------------------------------------------------------

def stored(fp8, x, scale, group, pad=None, offset=0):
    """8-bit rows of x inside a buffer of NaN codes: rows at a stride of `pad`, `offset` bytes in."""
    r = fp8.quantize(x, scale=scale, group=group)
    if pad is None:
        return r
    rows, dim = x.shape
    buffer = torch.full((rows * pad + offset + 64,), 0x7f, dtype=torch.uint8, device="cuda")
    codes = torch.as_strided(buffer, (rows, dim), (pad, 1), offset)
    codes.copy_(r.codes.view(torch.uint8))
    return fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), r.scales, group)


def check_product(a, b, got):
    x, y = values(a), values(b)
    want = x @ y.t()
    dim = x.shape[1]
    # sums in 32 bits: one rounding or truncation (2^-23) for each of dim products and additions, three more a block for its
    # scales; then half a step of the result's type, and for float16 half its smallest step
    sums = x.abs() @ y.abs().t()
    bound = (2 * dim + 3 * (-(-dim // 128))) * 2.0 ** -23 * sums + 2.0 ** -126
    if got.dtype != torch.float32:
        # the 8-bit matrix instructions add products in groups of eight, each cut off at 2^-13 of the largest: seven may lose that much
        bound = bound + 7 * 2.0 ** -13 * sums
    step = torch.finfo(got.dtype).eps / 2
    bound = bound + (want.abs() + bound) * step + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    over = want.abs() > torch.finfo(got.dtype).max
    off = (got.double() - want).abs()
    assert bool(((off <= bound) | over).all()), float((off / bound).max())


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("e8m0", 128), ("f32", 128)])
@pytest.mark.parametrize("dim", [1, 8, 16, 100, 127, 128, 129, 200, 256, 384, 520, 1000, 1536])
def test_matmul(fp8, scale, group, dim):
    for i, (m, n) in enumerate([(1, 1), (1, 300), (3, 65), (16, 128), (17, 257), (33, 15), (65, 130), (128, 64), (130, 127), (257, 300), (300, 1)]):
        a = fp8.quantize(torch.randn(m, dim, generator=gen(i), device="cuda"), scale=scale)
        b = fp8.quantize(torch.randn(n, dim, generator=gen(100 + i), device="cuda") * torch.exp2(torch.arange(n, device="cuda") % 7 - 3.0)[:, None], scale=scale, group=group)
        check_product(a, b, fp8.matmul(a, b, dtype=DTYPES[i % 3]))


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 128)])
@pytest.mark.parametrize("m,n,dim", [(1, 5000, 4096), (256, 1000, 2048), (512, 777, 1111), (1024, 1024, 640), (1000, 3000, 128), (2049, 515, 384)])
def test_matmul_larger(fp8, scale, group, m, n, dim):
    a = fp8.quantize(torch.randn(m, dim, generator=gen(7), device="cuda"), scale=scale)
    b = fp8.quantize(torch.randn(n, dim, generator=gen(8), device="cuda"), scale=scale, group=group)
    for dtype in DTYPES:
        check_product(a, b, fp8.matmul(a, b, dtype=dtype))


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("e8m0", 128), ("f32", 128)])
@pytest.mark.parametrize("m,n,dim", [(17, 130, 200), (31, 1000, 129), (32, 4097, 256), (33, 140_000, 128), (64, 70_003, 130), (129, 45_000, 256), (192, 23_000, 40), (250, 20_001, 384)])
def test_matmul_narrow_tiles(fp8, scale, group, m, n, dim):
    """Sizes that go to tiles of 32 or 64 rows of a by 128 of b."""
    a = fp8.quantize(torch.randn(m, dim, generator=gen(15), device="cuda"), scale=scale)
    b = fp8.quantize(torch.randn(n, dim, generator=gen(16), device="cuda") * torch.exp2(torch.arange(n, device="cuda") % 5 - 2.0)[:, None], scale=scale, group=group)
    for dtype in DTYPES:
        check_product(a, b, fp8.matmul(a, b, dtype=dtype))


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("f32", 128)])
@pytest.mark.parametrize("m,n,dim", [(16, 300, 3900), (16, 300, 4096), (16, 4097, 8192), (15, 700, 8900), (16, 130, 9500), (8, 100, 16384), (9, 100, 16384), (3, 8200, 16384), (4, 8200, 16384)])
def test_matmul_few_long_rows(fp8, scale, group, m, n, dim):
    """Few rows of a as long as fit a compute unit's memory, and longer."""
    a = fp8.quantize(torch.randn(m, dim, generator=gen(13), device="cuda"), scale=scale)
    b = fp8.quantize(torch.randn(n, dim, generator=gen(14), device="cuda"), scale=scale, group=group)
    for dtype in DTYPES:
        check_product(a, b, fp8.matmul(a, b, dtype=dtype))


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("f32", 128)])
@pytest.mark.parametrize("dim,pad,offset", [(256, 272, 0), (256, 256, 4), (256, 257, 0), (200, 208, 0), (200, 201, 3), (1000, 1008, 0), (129, 130, 1), (100, 4096, 16)])
@pytest.mark.parametrize("m,n", [(2, 70), (70, 300), (300, 290)])
def test_matmul_strided(fp8, scale, group, dim, pad, offset, m, n):
    """Codes at odd places and strides with NaN codes between the rows, results inside a wider buffer: nothing else changes."""
    a = stored(fp8, torch.randn(m, dim, generator=gen(9), device="cuda"), scale, 1, pad, offset)
    b = stored(fp8, torch.randn(n, dim, generator=gen(10), device="cuda"), scale, group, pad, offset)
    for dtype in DTYPES:
        buffer = torch.full((m + 2, n + 5), -7.0, dtype=dtype, device="cuda")
        out = buffer[1:-1, 3:-2]
        assert fp8.matmul(a, b, out=out) is out
        check_product(a, b, out)
        out.fill_(-7.0)
        assert bool((buffer == -7.0).all())


def test_matmul_shared_and_strided_scales(fp8):
    """Scales inside a wider buffer, and one row of a seen many times (stride 0)."""
    x, y = torch.randn(1, 300, generator=gen(11), device="cuda"), torch.randn(200, 300, generator=gen(12), device="cuda")
    for scale, group in (("e8m0", 1), ("f32", 128), ("e8m0", 128)):
        a, b = fp8.quantize(x, scale=scale), fp8.quantize(y, scale=scale, group=group)
        wide = torch.zeros(b.scales.shape[0], 9, dtype=torch.uint8 if scale == "e8m0" else torch.float32, device="cuda")
        wide[:, 2:5] = b.scales.view(wide.dtype)
        b2 = fp8.Fp8Rows(b.codes, wide.view(b.scales.dtype)[:, 2:5], group)
        a2 = fp8.Fp8Rows(a.codes.expand(40, -1), a.scales.view(wide.dtype).expand(40, -1).view(a.scales.dtype), 1)
        one, many = fp8.matmul(a, b), fp8.matmul(a2, b2)
        check_product(a2, b2, many)
        check_product(a, b, one)


@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
def test_matmul_nan_stays_in_its_row(fp8, scale, m):
    x, y = torch.randn(m, 300, generator=gen(13), device="cuda"), torch.randn(280, 300, generator=gen(14), device="cuda")
    x[m // 2, 290] = float("nan")
    y[40, 5] = float("inf")
    a, b = fp8.quantize(x, scale=scale), fp8.quantize(y, scale=scale)
    got = torch.isnan(fp8.matmul(a, b))
    want = torch.zeros_like(got)
    want[m // 2] = True
    want[:, 40] = True
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 200])
def test_matmul_every_scale_byte(fp8, dtype, m):
    """Products of each e8m0 scale, the smallest and NaN among them, with one that brings it near 1."""
    scale = torch.arange(256, device="cuda", dtype=torch.uint8)
    codes = torch.randint(0, 256, (256, 128), generator=gen(15), device="cuda").to(torch.uint8)
    codes[(codes & 0x78) < 0x30] = 0x38                    # magnitudes of 1/2 and more: normal numbers whatever the scale
    codes[(codes & 0x7f) == 0x7f] = 0x3c
    b = fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), scale[:, None].view(torch.float8_e8m0fnu))
    for e in (0, 1, 60, 127, 200, 254):
        a = fp8.Fp8Rows(codes[:1].expand(m, -1).contiguous().view(torch.float8_e4m3fn), torch.full((m, 1), e, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))
        got = fp8.matmul(a, b, dtype=dtype)
        assert bool(torch.isnan(got[:, 255]).all())
        near = (scale.long() + e - 254 > -90) & (scale.long() + e - 254 < 90) & (scale.long() > 1) & (scale.long() < 240) & (torch.tensor(1 < e < 240, device="cuda"))
        if dtype == torch.float16:
            near &= (scale.long() + e - 254 > -20) & (scale.long() + e - 254 < -10)
        if bool(near.any()):
            check_product(a, fp8.Fp8Rows(b.codes[near], b.scales.view(torch.uint8)[near].view(torch.float8_e8m0fnu)), got[:, near])


def test_matmul_zero_scales_and_extremes(fp8):
    """Rows of zeros, the smallest and the largest scales: products that leave 32 bits at either end."""
    x = torch.zeros(5, 256, device="cuda")
    x[1] = 1e-38
    x[2] = 1e30
    x[3] = 1e8
    x[4, 0] = 1.0
    for scale in ("e8m0", "f32"):
        r = fp8.quantize(x, scale=scale)
        got = fp8.matmul(r, r)
        assert bool((got[0] == 0).all()) and bool((got[:, 0] == 0).all())
        assert torch.isinf(got[2, 2]) and float(got[1, 1]) == 0.0
        check_product(r, r, torch.where(torch.isinf(got), 3.0e38, got))


# ---- rescore --------------------------------------------------------------------------------------

def plain_rescore(queries, rows, slots, k):
    v, n = values(rows).cpu().numpy(), len(rows)
    q, slots = queries.double().cpu().numpy(), slots.cpu().numpy()
    out_s, out_i = np.full((len(q), k), -np.inf, np.float32), np.full((len(q), k), -1, np.int64)
    for r in range(len(q)):
        there = slots[r][(slots[r] >= 0) & (slots[r] < n)]
        s = (v[there] @ q[r]).astype(np.float32)
        order = np.lexsort((there, -s))[:k]
        out_s[r, :len(order)], out_i[r, :len(order)] = s[order], there[order]
    return out_s, out_i


def check_best(fp8, queries, rows, slots, k):
    s, i = fp8.rescore(queries, rows, slots, k)
    ws, wi = plain_rescore(queries, rows, slots, k)
    assert np.array_equal(i.cpu().numpy(), wi)
    s = s.cpu().numpy()
    fine = np.isfinite(ws)
    assert np.array_equal(s[~fine], ws[~fine])
    # sums in 64 bits, then one rounding to 32: the same value, or its neighbour where the sums fall on either side of a border
    assert bool((np.abs(s[fine] - ws[fine]) <= np.spacing(np.abs(ws[fine]))).all())


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("e8m0", 128), ("f32", 128)])
@pytest.mark.parametrize("dim", [1, 8, 100, 128, 200, 512, 1000, 1536])
def test_rescore(fp8, scale, group, dim):
    n = 500
    rows = fp8.quantize(torch.randn(n, dim, generator=gen(20), device="cuda"), scale=scale, group=group)
    for j, (nq, m, k) in enumerate([(1, 1, 1), (1, 100, 10), (3, 17, 17), (40, 33, 5), (7, 500, 100)]):
        q = torch.randn(nq, dim, generator=gen(21 + j), device="cuda").to(DTYPES[j % 3])
        slots = torch.randint(0, n, (nq, m), generator=gen(31 + j), device="cuda")
        check_best(fp8, q, rows, slots, k)


@pytest.mark.parametrize("m,k", [(1000, 1), (1025, 1025), (5000, 30), (16384, 100)])
def test_rescore_many_candidates(fp8, m, k):
    rows = fp8.quantize(torch.randn(20000, 64, generator=gen(40), device="cuda"))
    q = torch.randn(2, 64, generator=gen(41), device="cuda")
    check_best(fp8, q, rows, torch.randint(0, 20000, (2, m), generator=gen(42), device="cuda"), k)


@pytest.mark.parametrize("nq,m", [(1, 128), (1, 129), (127, 129), (128, 129), (128, 256), (128, 257), (256, 40), (257, 40), (257, 256), (300, 257)])
@pytest.mark.parametrize("dim", [96, 2000])
def test_rescore_where_the_forms_meet(fp8, nq, m, dim):
    """Numbers of queries and candidates on both sides of where a call takes two launches, and a query fewer waves."""
    rows = fp8.quantize(torch.randn(700, dim, generator=gen(51), device="cuda"))
    q = torch.randn(nq, dim, generator=gen(52), device="cuda")
    slots = torch.randint(-3, 703, (nq, m), generator=gen(53), device="cuda")
    check_best(fp8, q, rows, slots, min(m, 30))


@pytest.mark.parametrize("dim,pad,offset", [(256, 257, 0), (200, 201, 3), (16384, 16384, 0), (10000, 10000, 0)])
def test_rescore_odd_places_and_long_rows(fp8, dim, pad, offset):
    rows = stored(fp8, torch.randn(50, dim, generator=gen(43), device="cuda"), "e8m0", 1, pad, offset)
    base = torch.randn(4, dim + 5, generator=gen(44), device="cuda")
    slots = torch.randint(0, 50, (4, 60), generator=gen(45), device="cuda")
    check_best(fp8, base[:, 3:3 + dim], rows, slots[:, 7:40], 9)


def test_rescore_absent_and_repeated(fp8):
    """Slots outside the rows, the same slot twice, rows of equal scores, queries with fewer candidates than k, and with none."""
    x = torch.randn(64, 128, generator=gen(46), device="cuda")
    x[10:20] = x[10]
    rows = fp8.quantize(x)
    slots = torch.randint(0, 64, (5, 30), generator=gen(47), device="cuda")
    slots[0, :5] = torch.tensor([-1, 64, 2 ** 40, -2 ** 62, 63], device="cuda")
    slots[1] = -1
    slots[2, :10] = torch.arange(19, 9, -1, device="cuda")
    slots[3] = 7
    slots[4, 3:] = 1 << 31
    check_best(fp8, torch.randn(5, 128, generator=gen(48), device="cuda"), rows, slots, 30)
    check_best(fp8, torch.zeros(5, 128, device="cuda"), rows, slots, 12)
    empty = fp8.Fp8Rows(rows.codes[:0], rows.scales[:0])
    s, i = fp8.rescore(torch.randn(5, 128, device="cuda"), empty, slots, 3)
    assert bool(torch.isinf(s).all()) and bool((i == -1).all())


def test_rescore_nan_comes_last(fp8):
    x = torch.randn(20, 130, generator=gen(49), device="cuda")
    x[3, 129] = float("nan")
    rows = fp8.quantize(x)
    slots = torch.arange(20, device="cuda")[None]
    s, i = fp8.rescore(torch.randn(1, 130, generator=gen(50), device="cuda"), rows, slots, 20)
    assert int(i[0, 19]) == 3 and bool(torch.isnan(s[0, 19])) and not bool(torch.isnan(s[0, :19]).any())


# ---- how calls run ----------------------------------------------------------------------------------

def test_on_another_stream_and_in_a_graph(fp8):
    """Each call on a stream of the caller's, and recorded: every replay gives what a call gives, with other inputs in the same
    buffers, other work between them and two graphs taken in turn."""
    q = torch.randn(70, 512, generator=gen(60), device="cuda")
    rows = fp8.quantize(torch.randn(1000, 512, generator=gen(61), device="cuda"))
    slots = torch.randint(0, 1000, (70, 40), generator=gen(62), device="cuda")

    def everything(n):
        a = fp8.quantize(q[:n])
        return (a.codes.view(torch.uint8), a.scales.view(torch.uint8), fp8.matmul(a, rows)) + fp8.rescore(q[:n], rows, slots[:n], 8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = everything(70)
    with torch.cuda.stream(side):
        got = everything(70)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graphs = []
    for n in (70, 3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = everything(n)
        graphs.append((n, graph, held))
    for turn in range(3):
        q.copy_(torch.randn(70, 512, generator=gen(70 + turn), device="cuda"))
        for n, graph, held in graphs:
            graph.replay()
            torch.randn(100_000, device="cuda").sum().item()
            assert all(torch.equal(x, y) for x, y in zip(everything(n), held))


def test_search_then_rescore_then_product(fp8):
    """As a service would: 2-bit codes find candidates, 8-bit rows put them in order; the product over all rows agrees."""
    from turbovec_amd import _lib as T
    n, dim, nq, m, k = 20000, 256, 9, 100, 10
    x = torch.nn.functional.normalize(torch.randn(n, dim, generator=gen(80), device="cuda"))
    q = torch.nn.functional.normalize(x[:nq] + 0.02 * torch.randn(nq, dim, generator=gen(81), device="cuda"))
    ix = T.NativeIndex(dim, 2)
    torch.cuda.synchronize()
    ix.add_dev(x.data_ptr(), n)
    scores, slots = torch.empty(nq, m, device="cuda"), torch.empty(nq, m, dtype=torch.int64, device="cuda")
    assert ix.search_dev(q.data_ptr(), nq, m, scores.data_ptr(), slots.data_ptr()) == m
    rows = fp8.quantize(x)
    s, best = fp8.rescore(q, rows, slots, k)
    check_best(fp8, q, rows, slots, k)
    assert bool((best[:, 0] == torch.arange(nq, device="cuda")).all())
    a = fp8.quantize(q)
    full = fp8.matmul(a, rows)
    check_product(a, rows, full)
    assert bool((full.argmax(1) == torch.arange(nq, device="cuda")).all())
    ix.close()


def test_a_buffer_past_four_gigabytes(fp8):
    """Rows and results whose offsets pass 32 bits."""
    n, dim = 33_000, 16384 * 8
    buffer = torch.zeros(n, dim, dtype=torch.uint8, device="cuda")          # 4.3 GB; rows are 256 of each 131072 codes
    x = torch.randn(n, 256, generator=gen(90), device="cuda")
    r = fp8.quantize(x)
    buffer[:, :256] = r.codes.view(torch.uint8)
    far = fp8.Fp8Rows(buffer.view(torch.float8_e4m3fn)[:, :256], r.scales)
    for m in (2, 100):
        a = fp8.quantize(torch.randn(m, 256, generator=gen(91), device="cuda"))
        assert torch.equal(fp8.matmul(a, far), fp8.matmul(a, r))
    slots = torch.randint(32_000, n, (3, 50), generator=gen(92), device="cuda")
    for x, y in zip(fp8.rescore(x[:3], far, slots, 9), fp8.rescore(x[:3], r, slots, 9)):
        assert torch.equal(x, y)


def test_more_rows_and_queries_than_a_grid_has(fp8):
    """Numbers of rows and queries for which workgroups go round: each part gives what it gives in a call of its own."""
    x = torch.randn(34_000_000, 1, generator=gen(93), device="cuda")
    for group in (1, 128):
        r = fp8.quantize(x, group=group)
        for lo in (0, 33_553_408, 33_999_872 - 128):
            part = fp8.quantize(x[lo:lo + 128], group=group)
            assert torch.equal(r.codes[lo:lo + 128].view(torch.uint8), part.codes.view(torch.uint8))
            assert torch.equal(r.scales[lo // group:lo // group + len(part.scales)].view(torch.uint8), part.scales.view(torch.uint8))
    del x, r
    rows = fp8.quantize(torch.randn(500, 40, generator=gen(94), device="cuda"))
    q = torch.randn(70_000, 40, generator=gen(95), device="cuda")
    for m in (3, 300):
        slots = torch.randint(0, 500, (70_000, m), generator=gen(96), device="cuda")
        got = fp8.rescore(q, rows, slots, 3)
        for lo in (0, 65_500, 69_900):
            for a, b in zip(got, fp8.rescore(q[lo:lo + 100], rows, slots[lo:lo + 100], 3)):
                assert torch.equal(a[lo:lo + 100], b)


# ---- scales far from 1 -----------------------------------------------------------------------------

# (each sum of rows of b, tiles of 32, 64, 128 and 256, rows of a in LDS)
FAR_SIZES = [(1, 300), (5, 40), (16, 17_000), (20, 300), (70, 300), (64, 70_000), (1000, 3000), (129, 45_000)]


def check_far(a, b, got):
    """Like check_product, but nothing is lost to subnormal numbers other than the result's own."""
    x, y = values(a), values(b)
    want, sums = x @ y.t(), x.abs() @ y.abs().t()
    dim, blocks = x.shape[1], -(-x.shape[1] // 128)
    step = torch.finfo(got.dtype).eps / 2
    # sums in 32 bits, as in check_product; a rounding of each block's sum and of each addition to the smallest 32-bit number, 2^-149, the former
    # times what is left of the scales when powers of two have been taken out, no more than 2^2 where such a sum is that small; half the result type's own
    bound = (2 * dim + 3 * blocks) * 2.0 ** -23 * sums + 8 * blocks * 2.0 ** -149 + (0 if got.dtype == torch.float32 else 7 * 2.0 ** -13) * sums
    bound = bound + (want.abs() + bound) * step + torch.finfo(got.dtype).smallest_normal * step
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("scale,group", [("f32", 1), ("f32", 128), ("e8m0", 1)])
@pytest.mark.parametrize("m,n", FAR_SIZES)
def test_matmul_products_of_scales_that_32_bits_do_not_hold(fp8, scale, group, m, n):
    """Tiny rows on both sides, whose products are numbers though the products of their scales are not."""
    x, y = torch.randn(m, 300, generator=gen(200), device="cuda"), torch.randn(n, 300, generator=gen(201), device="cuda")
    for size in (1e-17, 1e-18, 1e-19, 1e-20):
        a, b = fp8.quantize(x * size, scale=scale), fp8.quantize(y * size, scale=scale, group=group)
        for dtype in (torch.float32, torch.bfloat16):
            got = fp8.matmul(a, b, dtype=dtype)
            check_far(a, b, got)
            assert size < 1e-19 or bool((got.abs() > 1e-40).any())


@pytest.mark.parametrize("scale,group", [("f32", 1), ("f32", 128), ("e8m0", 1)])
@pytest.mark.parametrize("m,n", FAR_SIZES)
def test_matmul_of_huge_rows_that_do_not_meet(fp8, scale, group, m, n):
    """Coordinates of which one factor is 0 everywhere: 0, however large the scales are."""
    for size in (1e10, 1e22, 1e23, 1e30, 1e33):
        x, y = torch.zeros(m, 300, device="cuda"), torch.zeros(n, 300, device="cuda")
        x[:, ::2], y[:, 1::2] = size, -size
        a, b = fp8.quantize(x, scale=scale), fp8.quantize(y, scale=scale, group=group)
        for dtype in DTYPES:
            assert bool((fp8.matmul(a, b, dtype=dtype) == 0).all()), (size, dtype)


@pytest.mark.parametrize("scale,group", [("f32", 1), ("f32", 128), ("e8m0", 1), ("e8m0", 128)])
@pytest.mark.parametrize("m,n", FAR_SIZES)
def test_matmul_of_scales_that_make_up_for_each_other(fp8, scale, group, m, n):
    """Blocks whose scale is far above 1 on one side and as far below on the other: each counts as much as the next."""
    dim = 128 * 12 + 40
    power = torch.tensor([0, 60, -60, 63, -63, 64, -64, 65, -65, 90, -90, 102, -102], device="cuda").float()

    def rows(count, group, sign, seed):
        codes = torch.randint(0, 256, (count, dim), generator=gen(seed), device="cuda").to(torch.uint8)
        codes[(codes & 0x7f) == 0x7f] = 0x3c
        s = torch.exp2(sign * power).repeat(-(-count // group), 1)
        if scale == "f32":
            s *= 1 + 0.99 * torch.rand(s.shape, generator=gen(seed + 1), device="cuda")
            return fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), s, group)
        bytes_ = (127 + sign * power).to(torch.uint8).repeat(len(s), 1)
        return fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), bytes_.view(torch.float8_e8m0fnu), group)

    a, b = rows(m, 1, 1, 210), rows(n, group, -1, 220)
    for dtype in (torch.float32, torch.bfloat16):
        check_far(a, b, fp8.matmul(a, b, dtype=dtype))


@pytest.mark.parametrize("group", [1, 128])
@pytest.mark.parametrize("m,n", FAR_SIZES)
def test_matmul_scales_that_are_no_numbers(fp8, group, m, n):
    """A scale of b that is infinite or NaN, negative, 0, or the smallest and the largest there are."""
    codes = lambda rows, seed: (torch.randint(0x28, 0x48, (rows, 256), generator=gen(seed), device="cuda")).to(torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    inf, nan, tiny = float("inf"), float("nan"), 2.0 ** -149
    sa = torch.ones(m, 2, device="cuda")
    sb = torch.ones(-(-n // group), 2, device="cuda")
    sb[0, 1] = nan
    if len(sb) > 2:
        sb[1, 0], sb[2, 0] = inf, -3.0
    if len(sb) > 20:
        sb[3], sb[4], sb[5] = 0.0, tiny, 1e-10
    a, b = fp8.Fp8Rows(codes(m, 230), sa), fp8.Fp8Rows(codes(n, 231), sb, group)
    for dtype in (torch.float32, torch.bfloat16):
        got = fp8.matmul(a, b, dtype=dtype)
        row = torch.arange(n, device="cuda") // group
        assert bool(torch.isnan(got[:, row == 0]).all())
        if len(sb) > 2:
            assert bool((got[:, row == 1] == inf).all())
        plain = (row != 0) & ((row != 1) | (len(sb) <= 2))
        if bool(plain.any()):
            check_far(a, fp8.Fp8Rows(b.codes[plain], sb[row[plain]]), got[:, plain])
    for x, y in ((2.0 ** 103, tiny), (2.0 ** -108, 3.4e38)):
        x, y = fp8.Fp8Rows(a.codes, torch.full_like(sa, x)), fp8.Fp8Rows(b.codes, torch.full_like(sb, y), group)
        check_far(x, y, fp8.matmul(x, y))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n_scales", [(1, 255), (40, 255), (300, 255)])
def test_matmul_scale_bytes_at_both_ends(fp8, dtype, m, n_scales):
    """Every e8m0 scale against those at either end and in between, wherever the products are ordinary numbers.  32-bit results take coordinates as numbers that
    32 bits hold: 448 * 2^119, byte 246, is the last that they do."""
    codes = torch.randint(0, 256, (n_scales, 128), generator=gen(240), device="cuda").to(torch.uint8)
    codes[(codes & 0x78) < 0x30] = 0x38                    # magnitudes of 1/2 and more: their last bit is 2^-4, times 2^-127 a number of bfloat16
    codes[(codes & 0x7f) == 0x7f] = 0x3e
    codes[:, 0] = 0x7e                                     # 448
    scale = torch.arange(n_scales, device="cuda", dtype=torch.uint8)
    b = fp8.Fp8Rows(codes.view(torch.float8_e4m3fn), scale[:, None].view(torch.float8_e8m0fnu))
    compared = torch.zeros(n_scales, dtype=torch.bool, device="cuda")
    for e in (0, 1, 2, 3, 20, 127, 235, 245, 246, 247, 253, 254):
        a = fp8.Fp8Rows(codes[7:8].expand(m, -1).contiguous().view(torch.float8_e4m3fn), torch.full((m, 1), e, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))
        got = fp8.matmul(a, b, dtype=dtype)
        held = (scale <= 246) & (e <= 246) if dtype == torch.float32 else scale <= 254
        near = ((scale.long() + e - 254).abs() < 100) & held
        compared |= near
        if bool(near.any()):
            check_far(a, fp8.Fp8Rows(b.codes[near], scale[near][:, None].view(torch.float8_e8m0fnu)), got[:, near])
        assert bool(near.any()) or (dtype == torch.float32 and e > 246)
        if dtype == torch.float32:
            assert not bool(torch.isfinite(got[:, ~held]).any())
    assert bool(compared[:247].all()) and (dtype == torch.float32 or bool(compared.all()))


# ---- what sums lose --------------------------------------------------------------------------------

def root_mean_square(x):
    return float(x.pow(2).mean().sqrt())


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("f32", 128)])
@pytest.mark.parametrize("m,n,dim", [(4, 3000, 200), (4, 3000, 1536), (20, 1000, 1536), (70, 600, 384), (1030, 1000, 1536)])
def test_matmul_32_bit_results_lose_what_32_bit_sums_do(fp8, scale, group, m, n, dim):
    """Of random rows.  `dim` roundings, 2^-24 at most of a running sum that is no larger than the result on average, and half of them either way; three a block for the
    scales.  (Products cut off as those of 16-bit results are would make it 1.4e-5.)"""
    a = fp8.quantize(torch.randn(m, dim, generator=gen(250), device="cuda"), scale=scale)
    b = fp8.quantize(torch.randn(n, dim, generator=gen(251), device="cuda"), scale=scale, group=group)
    want = values(a) @ values(b).t()
    off = root_mean_square(fp8.matmul(a, b).double() - want) / root_mean_square(want)
    assert off <= 2.0 ** -24 * (dim + 3 * -(-dim // 128)) ** 0.5, off


@pytest.mark.parametrize("scale,group", [("e8m0", 1), ("f32", 1), ("f32", 128)])
@pytest.mark.parametrize("m,n,dim", [(4, 3000, 200), (4, 3000, 1536), (70, 600, 384), (130, 300, 1536), (500, 300, 1000)])
def test_matmul_16_bit_results_lose_what_is_said(fp8, scale, group, m, n, dim):
    """Products are added in groups of eight neighbours, each cut off, towards zero, at 2^-13 of the group's largest, whose factors count as the powers of two
    at or below them: 1.4e-5 of the usual result, seen where results are small, so that rounding them loses less."""
    a = fp8.quantize(torch.randn(m, dim, generator=gen(252), device="cuda"), scale=scale)
    b = fp8.quantize(torch.randn(n, dim, generator=gen(253), device="cuda"), scale=scale, group=group)
    want = values(a) @ values(b).t()
    power = lambda v: torch.where(v == 0, -100.0, torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -9))))  # noqa: E731
    said = torch.zeros_like(want)
    sb = b.scales.double().repeat_interleave(group, 0)[:n]
    for k in range(0, dim, 8):
        x, y = a.codes[:, k:k + 8].double(), b.codes[:, k:k + 8].double()
        at = torch.exp2((power(x)[:, None] + power(y)[None]).amax(2, keepdim=True) - 13)
        said += (torch.trunc(x[:, None] * y[None] / at) * at).sum(2) * a.scales[:, k // 128, None].double() * sb[None, :, k // 128]
    size = root_mean_square(want)
    small = want.abs() < size / 64
    got = fp8.matmul(a, b, dtype=torch.float16).double()
    off = root_mean_square((got - said)[small]) / size
    # half a step of float16 of 1/64 of the size and of what is cut off, 2^-13 of a product at most; and of sums of groups and blocks 2^-23 each
    assert off <= 2.0 ** -11 * (1 / 64 + 2.0 ** -13) + 2.0 ** -23 * (dim / 8 + 2 * -(-dim // 128)) ** 0.5, off


def test_the_documented_path_from_an_index(fp8):
    """Numpy slots of a TurboQuantIndex to re-scoring, a mask packed for it to a draw, and rows that move as its slots do."""
    from turbovec_amd import _lib as T
    from turbovec_amd.index import TurboQuantIndex
    from turbovec_amd.sampling import sample
    n, dim, nq = 3000, 200, 6
    x = torch.nn.functional.normalize(torch.randn(n, dim, generator=gen(260), device="cuda"))
    queries = torch.nn.functional.normalize(x[-nq:] + 0.02 * torch.randn(nq, dim, generator=gen(261), device="cuda"))
    index, rows = TurboQuantIndex(dim, 4), fp8.quantize(x)
    index.add(x.cpu().numpy())

    def look():
        slots = torch.from_numpy(index.search(queries.cpu().numpy(), 50)[1]).cuda()
        check_best(fp8, queries, rows, slots, 10)
        return fp8.rescore(queries, rows, slots, 10)[1]

    assert torch.equal(look()[:, 0], torch.arange(n - nq, n, device="cuda"))
    allowed = np.zeros(n, bool)
    allowed[n - nq:] = allowed[5] = True
    words = torch.from_numpy(T.pack_mask(allowed)[0].view(np.int64)).cuda()
    drawn, probs = sample(fp8.matmul(fp8.quantize(queries), rows), torch.rand(nq, generator=gen(262), device="cuda"), temperature=1e-3, mask=words)
    assert torch.equal(drawn, torch.arange(n - nq, n, device="cuda")) and bool((probs > 0.99).all())
    for slot in (17, n - nq - 2, n - 2 - 2, 0):
        last = index.swap_remove(slot)
        rows.codes.view(torch.uint8)[slot] = rows.codes.view(torch.uint8)[last]
        rows.scales.view(torch.uint8)[slot] = rows.scales.view(torch.uint8)[last]
        rows = fp8.Fp8Rows(rows.codes[:last], rows.scales[:last])
        x[slot] = x[last]
        x = x[:last]
        assert torch.equal(look()[:, 0], (queries @ x.t()).argmax(1))
