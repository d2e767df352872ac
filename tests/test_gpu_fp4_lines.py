"""Products whose result's rows start at whole cache lines, in their middle and elsewhere: the same numbers, and nothing beside them."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("m,n,dim", [(1000, 5000, 768), (300, 20_011, 512), (130, 9000, 1536), (257, 7777, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_where_rows_start(m, n, dim, dtype):
    from turbovec_amd import fp4
    g = torch.Generator(device="cuda").manual_seed(m)
    a, b = (fp4.quantize(torch.randn(rows, dim, generator=g, device="cuda")) for rows in (m, n))
    want = fp4.matmul(a, b, dtype=dtype)
    line = 128 // want.element_size()
    for stride in (-(-n // line) * line, -(-n // line) * line + line // 2, -(-n // line) * line + 3):
        for off in (0, line // 2, 1):
            buffer = torch.full((m * stride + 2 * line,), 7.0, dtype=dtype, device="cuda")
            out = torch.as_strided(buffer, (m, n), (stride, 1), off)
            assert fp4.matmul(a, b, out=out) is out
            assert torch.equal(out, want)
            out.fill_(7.0)
            assert bool((buffer == 7).all())
