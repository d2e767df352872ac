"""Norms that end in 8- or 4-bit rows, against the formula in 64 bits."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
KINDS = [("fp8", "e8m0"), ("fp8", "f32"), ("fp4", "e8m0")]
EPS = 1e-6


@pytest.fixture(scope="module")
def norm():
    from turbovec_amd import norm
    return norm


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(rows, dim, dtype, seed=1):
    g = gen(seed)
    spread = torch.exp(torch.randn(dim, generator=g, device="cuda"))
    x, r = ((s * spread * torch.randn(rows, dim, generator=g, device="cuda")).to(dtype) for s in (1, 3))
    return x, r, 1 + 0.3 * torch.randn(dim, generator=g, device="cuda")


def row_values(rows):
    if hasattr(rows, "values"):
        return rows.values().double()
    return rows.codes.double() * rows.scales.double().repeat_interleave(128, 1)[:, :rows.dim]


def check(rows, h, weight, to, scale, eps=EPS):
    """`h` in 64 bits.  The kernel's y: h is rounded (2^-24 of it), squares are added one after the other along a thread and then by halves, at most 64 + 16 roundings of
    2^-24, half of which reach the root; the mean, eps, root, quotient, two products: 8 more.  Codes: half a step of what the code holds beside that; a scale may lie as
    far from the exact one, and one power of two beside it only where the maximum is that near to the border."""
    off = (1 + 40 + 8) * 2.0 ** -24
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * (1.0 if weight is None else weight.double())
    block, top = (32, 7.0) if to == "fp4" else (128, 448.0)
    count, dim = y.shape
    padded = torch.nn.functional.pad(y.abs(), (0, -dim % block)).view(count, -1, block)
    most = padded.amax(2)
    s = rows.scales.double()
    if scale == "f32":
        assert bool(((s - (most / top).clamp(min=2.0 ** -126)).abs() <= s * (off + 2.0 ** -23)).all())
    else:
        least = s == 2.0 ** -126
        assert bool(((most <= top * s * (1 + off)).all()) and ((most >= top / 2 * s * (1 - off)) | least).all())
    wide = s.repeat_interleave(block, 1)[:, :dim]
    q = (y / wide).abs()
    if to == "fp4":
        half = torch.where(q < 2, 0.25, torch.where(q < 4, 0.5, 1.0))
    else:
        half = torch.clamp(torch.exp2(torch.floor(torch.log2(q.clamp(min=2.0 ** -40)))) * 2.0 ** -4, min=2.0 ** -10)
    off_by = (row_values(rows) - y).abs() / wide
    assert bool((off_by <= half * (1 + 1e-9) + 2 * off * q + 2.0 ** -100).all()), (off_by - half).max()


@pytest.mark.parametrize("rows,dim", [(1, 1), (2, 7), (3, 8), (5, 31), (4, 33), (3, 127), (4, 129), (70, 500), (33, 512), (9, 513), (130, 1000), (64, 2048), (5, 2049), (9, 4096), (4, 4104), (3, 8192),
                                      (5, 8200), (2, 16383), (3, 16384), (1000, 24), (4001, 130)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("to,scale", KINDS)
def test_norm(norm, rows, dim, dtype, to, scale):
    x, r, w = inputs(rows, dim, dtype)
    check(norm.rms_norm(x, eps=EPS, to=to, scale=scale), x.double(), None, to, scale)
    w = w.to(dtype)
    made, total = norm.add_rms_norm(x, r, w, eps=EPS, to=to, scale=scale)
    h = x.double() + r.double()
    check(made, h, w, to, scale)
    assert torch.equal(total, (x.float() + r.float()).to(dtype))                   # one rounding each


@pytest.mark.parametrize("x_type", DTYPES)
@pytest.mark.parametrize("w_type", DTYPES)
def test_weights_of_other_types(norm, x_type, w_type):
    x, _, w = inputs(20, 700, x_type)
    check(norm.rms_norm(x, w.to(w_type)), x.double(), w.to(w_type), "fp8", "e8m0", 1e-6)


@pytest.mark.parametrize("to,scale", KINDS)
@pytest.mark.parametrize("rows,dim", [(1, 4096), (37, 1000), (600, 333), (300, 4096), (4, 16384)])
def test_the_sum_takes_an_inputs_place(norm, to, scale, rows, dim):
    x, r, w = inputs(rows, dim, torch.bfloat16)
    want, total = norm.add_rms_norm(x, r, w, to=to, scale=scale)
    for place in ("x", "residual", "other"):
        a, b = x.clone(), r.clone()
        out = {"x": a, "residual": b, "other": torch.full_like(x, 3.0)}[place]
        made, got = norm.add_rms_norm(a, b, w, to=to, scale=scale, out=out)
        assert got is out and torch.equal(out, total)
        assert torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(made.scales.view(torch.uint8), want.scales.view(torch.uint8))
        assert place == "x" or torch.equal(a, x)
        assert place == "residual" or torch.equal(b, r)


@pytest.mark.parametrize("to,scale", KINDS)
def test_strided_and_beside_others(norm, to, scale):
    from turbovec_amd import _lib as T
    for off, dim in ((0, 256), (1, 300), (3, 97), (2, 2050)):
        x, r, w = inputs(40, dim + 9, torch.float16, 3)
        x, r, w = x[:, off:off + dim], r[:, off:off + dim], w[off:off + dim]
        want, total = norm.add_rms_norm(x.contiguous(), r.contiguous(), w.contiguous(), to=to, scale=scale)
        made, got = norm.add_rms_norm(x, r, w, to=to, scale=scale)
        assert torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(made.scales.view(torch.uint8), want.scales.view(torch.uint8)) and torch.equal(got, total)
        width, blocks = ((dim + 1) // 2, -(-dim // 32)) if to == "fp4" else (dim, -(-dim // 128))
        size = 4 if scale == "f32" else 1
        codes = torch.full((42, width + 13), 0x55, dtype=torch.uint8, device="cuda")
        scales = torch.full((42, blocks + 3, size), 0x55, dtype=torch.uint8, device="cuda")
        summed = torch.full((42, dim + 5), 9.0, dtype=torch.float16, device="cuda")
        T.check(T.lib().tv_rms_norm_dev(0, torch.cuda.current_stream().cuda_stream, x.data_ptr(), T.F16, x.stride(0), r.data_ptr(), r.stride(0), summed[1:].data_ptr() + 2 * off, dim + 5, w.data_ptr(), T.F32, 1e-6,
                                        40, dim, T.ROWS_FP4 if to == "fp4" else T.ROWS_FP8, T.SCALE_F32 if scale == "f32" else T.SCALE_E8M0, codes[1:].data_ptr() + off, width + 13, scales[1:].data_ptr(), blocks + 3))
        assert torch.equal(codes[1:41, off:off + width], want.codes.view(torch.uint8))
        assert torch.equal(scales[1:41, :blocks].reshape(40, -1), want.scales.view(torch.uint8).reshape(40, -1)) and torch.equal(summed[1:41, off:off + dim], total)
        codes[1:41, off:off + width], scales[1:41, :blocks], summed[1:41, off:off + dim] = 0x55, 0x55, 9.0
        assert bool((codes == 0x55).all()) and bool((scales == 0x55).all()) and bool((summed == 9).all())


@pytest.mark.parametrize("to,scale", KINDS)
@pytest.mark.parametrize("rows,dim", [(12, 300), (2000, 300), (12, 5000)])
def test_rows_that_are_no_numbers(norm, to, scale, rows, dim):
    """A row with a NaN or an infinity, one too large for its squares, and a row of zeros without eps are NaN; their neighbours are not."""
    x, _, _ = inputs(rows, dim, torch.float32)
    x[1, 5], x[3, dim - 1], x[5, 200], x[7], x[9] = float("nan"), float("inf"), 2.0 ** 80, 0.0, 1e-30
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[1, 3, 5]] = True
    made = norm.rms_norm(x, to=to, scale=scale)
    v = row_values(made)
    assert torch.equal(torch.isnan(v).all(1), bad) and torch.equal(torch.isnan(v).any(1), bad)
    assert bool((v[7] == 0).all())
    v = row_values(norm.rms_norm(x, to=to, scale=scale, eps=0))
    bad[[7, 9]] = True                                  # (1e-60 is 0 in 32 bits)
    assert torch.equal(torch.isnan(v).all(1), bad) and torch.equal(torch.isnan(v).any(1), bad)
    good = ~torch.tensor([i in (1, 3, 5, 7, 9) for i in range(rows)], device="cuda")
    assert torch.equal(v[good], row_values(norm.rms_norm(x[good].contiguous(), to=to, scale=scale, eps=0)))


@pytest.mark.parametrize("to,scale", KINDS)
def test_rows_do_not_depend_on_how_many_there_are(norm, to, scale):
    """The sums of a row go by its length alone."""
    for dim in (96, 1000, 4096, 6000):
        x, r, w = inputs(3000, dim, torch.bfloat16, 5)
        made, total = norm.add_rms_norm(x, r, w, to=to, scale=scale)
        for at, count in ((0, 1), (17, 5), (1000, 300)):
            some, part = norm.add_rms_norm(x[at:at + count], r[at:at + count], w, to=to, scale=scale)
            assert torch.equal(some.codes.view(torch.uint8), made.codes[at:at + count].view(torch.uint8)) and torch.equal(part, total[at:at + count])
            assert torch.equal(some.scales.view(torch.uint8), made.scales[at:at + count].view(torch.uint8))


def test_no_rows_and_many(norm):
    x = torch.randn(0, 64, device="cuda")
    assert len(norm.rms_norm(x)) == 0 and norm.add_rms_norm(x, x)[1].shape == (0, 64)
    x = torch.randn((1 << 22) + 77, 8, generator=gen(6), device="cuda", dtype=torch.float32).half()
    made = norm.rms_norm(x)
    check(norm.rms_norm(x[-1000:]), x[-1000:].double(), None, "fp8", "e8m0")
    assert torch.equal(made.codes[-1000:].view(torch.uint8), norm.rms_norm(x[-1000:]).codes.view(torch.uint8))


def test_refusals(norm):
    x = torch.zeros(4, 64, device="cuda")
    for call, kind, text in (
            (lambda: norm.rms_norm(x.t()), ValueError, "contiguous"),
            (lambda: norm.rms_norm(x, to="fp16"), ValueError, "to must be"),
            (lambda: norm.rms_norm(x, scale="e5m2"), ValueError, "scale must be"),
            (lambda: norm.rms_norm(x, to="fp4", scale="f32"), ValueError, "e8m0"),
            (lambda: norm.rms_norm(x, eps=-1), ValueError, "eps"),
            (lambda: norm.rms_norm(x, eps=float("nan")), ValueError, "eps"),
            (lambda: norm.rms_norm(x, torch.zeros(63, device="cuda")), ValueError, "weight must have 64"),
            (lambda: norm.rms_norm(x, torch.zeros(64)), ValueError, "weight must be on a GPU"),
            (lambda: norm.rms_norm(x, torch.zeros(64, device="cuda").double()), TypeError, "weight"),
            (lambda: norm.rms_norm(torch.zeros(2, 16385, device="cuda")), ValueError, "dim must be"),
            (lambda: norm.add_rms_norm(x, x.half()), TypeError, "residual"),
            (lambda: norm.add_rms_norm(x, x[:3]), ValueError, "residual must be"),
            (lambda: norm.add_rms_norm(x, x, out=x.half()), TypeError, "out"),
            (lambda: norm.add_rms_norm(x, x, out=x[:, :60]), ValueError, "out must be")):
        with pytest.raises(kind, match=text):
            call()


def test_on_another_stream_and_in_a_graph(norm):
    x, r, w = inputs(50, 1000, torch.bfloat16, 7)
    want, total = norm.add_rms_norm(x, r, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        made, got = norm.add_rms_norm(x, r, w)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got, total)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made, got = norm.add_rms_norm(x, r, w)
    for seed in (8, 9, 10):
        x.copy_(inputs(50, 1000, torch.bfloat16, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        want, total = norm.add_rms_norm(x, r, w)
        assert torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(made.scales.view(torch.uint8), want.scales.view(torch.uint8)) and torch.equal(got, total)


def test_a_buffer_past_four_gigabytes(norm):
    n, dim = 180_000, 64
    buffer = torch.empty(n * 12_000, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(buffer, (n, dim), (12_000, 1), 0)
    x, r, w = inputs(n, dim, torch.bfloat16, 11)
    far.copy_(x)
    want, total = norm.add_rms_norm(x, r, w)
    made, got = norm.add_rms_norm(far, r, w, out=far)
    assert torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got, total)


@pytest.mark.parametrize("to", ["fp8", "fp4"])
def test_norm_then_scores_then_a_draw_and_its_log_probability(norm, to):
    """A model's last step: the residual's sum, normed and quantised, scored against an output embedding's rows, a slot drawn and its log probability taken."""
    from turbovec_amd import fp4, fp8, sampling
    g = gen(12)
    q = fp8 if to == "fp8" else fp4
    table = q.quantize(torch.randn(5000, 512, generator=g, device="cuda"))
    x, r, w = inputs(9, 512, torch.bfloat16, 13)
    hidden, total = norm.add_rms_norm(x, r, w, to=to)
    scores = q.matmul(hidden, table) * 0.05
    want = (row_values(hidden) @ row_values(table).t()) * 0.05
    assert float((scores.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())
    slots, p = sampling.sample(scores, torch.rand(9, generator=g, device="cuda"), temperature=0.7)
    found = sampling.log_probs(scores, slots, temperature=0.7, top=5)
    z = torch.log_softmax(scores.double() / 0.7, 1)
    assert torch.allclose(found.log_probs.double(), z.gather(1, slots[:, None])[:, 0], atol=1e-4)
    assert torch.allclose(found.log_probs.exp(), p, rtol=1e-4, atol=0)
    assert torch.equal(found.top_slots, torch.sort(scores, dim=1, descending=True, stable=True).indices[:, :5])


def test_rows_that_are_one_and_the_same(norm):
    """An input may be one row many times, the sum may not."""
    one, other = torch.randn(1, 400, device="cuda"), torch.randn(7, 400, device="cuda")
    made, summed = norm.add_rms_norm(one.expand(7, 400), other)
    want, want_sum = norm.add_rms_norm(one.repeat(7, 1), other)
    assert torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(summed, want_sum)
    made, summed = norm.add_rms_norm(other, one.expand(7, 400), out=other)
    assert summed is other and torch.equal(other, want_sum) and torch.equal(made.codes.view(torch.uint8), want.codes.view(torch.uint8))
    with pytest.raises(RuntimeError, match="overlap"):
        norm.add_rms_norm(other, other, out=torch.zeros(1, 400, device="cuda").expand(7, 400))


@pytest.mark.parametrize("to", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [100, 512, 1536, 2048, 4096, 16384])
def test_scales_next_to_a_border(norm, dim, dtype, to):
    """Weights that bring each block's largest value next to where its power of two changes.  Of what the kernel decides by, the mean is off by what a thread's 8 or 16 squares lose in 32 bits, over
    many threads: by six standard deviations of sqrt(16) 2^-25 / sqrt(threads), half of which reaches the root; two products are off by 2^-24 each, but for 8-bit rows of 513 to 2048 two-byte values."""
    block, border = (32, 7.0) if to == "fp4" else (128, 448.0)
    threads = max(dim // 16, 6)
    off = 6 * 4 * 2.0 ** -25 / threads ** 0.5 / 2 + (0.0 if to == "fp8" and dtype == torch.bfloat16 and 512 < dim <= 2048 else 2 * 2.0 ** -24)
    told = 0
    for seed in range(60):
        g = gen(100 + seed)
        x = torch.randn(1, dim, generator=g, device="cuda").to(dtype)
        h = x.double()
        unit = h / torch.sqrt((h * h).mean() + EPS)
        weight = torch.full((dim,), 2.0 ** -9, device="cuda")
        best = torch.nn.functional.pad(unit.abs(), (0, -dim % block)).view(-1, block)
        at = best.argmax(1) + torch.arange(len(best), device="cuda") * block
        near = border * 2.0 ** torch.randint(-12, -8, (len(at),), generator=g, device="cuda").double() * (1 + 8 * off * (torch.rand(len(at), generator=g, device="cuda").double() - 0.5))
        weight[at] = (near / unit[0, at].abs()).float()
        most = torch.nn.functional.pad((unit * weight.double()).abs(), (0, -dim % block)).view(-1, block).amax(1)
        over = torch.log2(most / border)
        want = torch.floor(over) + 1 if to == "fp4" else torch.ceil(over)
        clear = ((over - torch.round(over)).abs() * 0.6931 > off) & (most > 0)
        got = torch.log2(norm.rms_norm(x, weight, eps=EPS, to=to).scales.double())[0]
        assert bool((got == want)[clear].all()), (seed, over[clear & (got != want)] - torch.round(over[clear & (got != want)]))
        assert bool(((got - over).abs() < 1.01).all())
        told += int((clear & ((over - torch.round(over)).abs() < 8 * off)).sum())
    assert told > 10
