"""Refusals of 4-bit rows, of norms that end in rows and of log probabilities, at the C ABI and in Python: no kernel is launched here and none would be."""
import pytest
import torch

from turbovec_amd import _lib as T
from turbovec_amd import fp4, fp8, norm, sampling

P = 4096                       # a place that is never read


def refused(rc, text):
    assert rc == T.ERR_BAD_ARGUMENT and text in T.lib().tv_last_error().decode(), T.lib().tv_last_error()


def quantize(device=0, x=P, x_type=T.F32, rows=4, dim=256, codes=P, code_stride=128, scales=P, scale_stride=8):
    return T.lib().tv_fp4_quantize_dev(device, None, x, x_type, dim, rows, dim, codes, code_stride, scales, scale_stride)


def values(codes=P, scales=P, rows=4, dim=256, out=P, out_type=T.F32, out_stride=256):
    return T.lib().tv_fp4_values_dev(0, None, codes, 128, scales, 8, rows, dim, out, out_type, out_stride)


def matmul(m=4, n=4, dim=256, a=P, a_scales=P, b=P, b_scales=P, out=P, out_type=T.F32, out_stride=4):
    return T.lib().tv_fp4_matmul_dev(0, None, a, 128, a_scales, 8, m, b, 128, b_scales, 8, n, dim, out, out_type, out_stride)


def rms_norm(x=P, x_type=T.BF16, x_stride=256, residual=None, residual_stride=256, total=None, sum_stride=256, weight=None, weight_type=T.F32, eps=1e-6, rows=4, dim=256,
             kind=T.ROWS_FP8, scale=T.SCALE_F32, codes=P, code_stride=256, scales=P, scale_stride=8):
    return T.lib().tv_rms_norm_dev(0, None, x, x_type, x_stride, residual, residual_stride, total, sum_stride, weight, weight_type, eps, rows, dim, kind, scale, codes, code_stride,
                                   scales, scale_stride)


def log_probs(scores=P, kind=T.F32, rows=2, n=100, mask=None, t=None, slots=P, given=1, top=3, lp=P, entropy=P, top_slots=P, top_lp=P, stats=None, ws=P, ws_bytes=1 << 40):
    return T.lib().tv_log_probs_dev(0, None, scores, kind, n, rows, n, mask, 0, t, slots, given, given, top, lp, entropy, top_slots, top_lp, stats, ws, ws_bytes)


def log_probs_grad(scores=P, kind=T.F32, rows=2, n=100, mask=None, t=None, slots=P, given=1, stats=P, g=P, ge=P, out=P, out_stride=100):
    return T.lib().tv_log_probs_grad_dev(0, None, scores, kind, n, rows, n, mask, 0, t, slots, given, given, stats, g, ge, out, out_stride)


@pytest.mark.parametrize("change,text", [
    (dict(dim=0), "dim"), (dict(dim=16385), "dim"), (dict(rows=1 << 31), "too many rows"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(x_type=3), "values"),
    (dict(x=None), "null"), (dict(x=P + 2), "aligned"), (dict(code_stride=127), "overlap"), (dict(scale_stride=7), "overlap"), (dict(dim=255, code_stride=127), "overlap")])
def test_quantize_refuses(change, text):
    refused(quantize(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(dim=0), "dim"), (dict(rows=1 << 31), "too many rows"), (dict(codes=None), "null"), (dict(out=None), "null"), (dict(out=P + 2), "aligned"), (dict(out_type=-1), "values"),
    (dict(out_stride=255), "overlap")])
def test_values_refuses(change, text):
    refused(values(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(dim=0), "dim"), (dict(dim=16385), "dim"), (dict(m=1 << 31), "rows"), (dict(n=1 << 31), "rows"), (dict(a=None), "null"), (dict(b=None), "null"), (dict(a_scales=None), "null"),
    (dict(b_scales=None), "null"), (dict(out=None), "null"), (dict(out=P + 2), "aligned"), (dict(out=P + 1, out_type=T.BF16), "aligned"), (dict(out_type=9), "values"), (dict(out_stride=3), "overlap")])
def test_matmul_refuses(change, text):
    refused(matmul(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(dim=0), "dim"), (dict(dim=16385), "dim"), (dict(rows=1 << 31), "too many rows"), (dict(kind=2), "kind"), (dict(kind=T.ROWS_FP4), "e8m0"), (dict(scale=2), "scales"), (dict(codes=None), "null"),
    (dict(scales=P + 2), "aligned"), (dict(x=None), "null"), (dict(x=P + 1), "aligned"), (dict(residual=P + 1), "aligned"), (dict(total=P + 1), "aligned"), (dict(weight=P + 2), "aligned"),
    (dict(weight=P, weight_type=3), "values"), (dict(x_type=3), "values"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(total=2 * P, sum_stride=255), "overlap"),
    (dict(total=P, sum_stride=300), "another stride"), (dict(residual=2 * P, total=2 * P, residual_stride=300), "another stride"), (dict(code_stride=255), "overlap"), (dict(scale_stride=1), "overlap"),
    (dict(kind=T.ROWS_FP4, scale=T.SCALE_E8M0, code_stride=127), "overlap"), (dict(kind=T.ROWS_FP4, scale=T.SCALE_E8M0, scale_stride=7), "overlap")])
def test_rms_norm_refuses(change, text):
    refused(rms_norm(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(n=0), "without scores"), (dict(n=1 << 31), "too many"), (dict(rows=1 << 31), "too many"), (dict(scores=None), "null"), (dict(scores=P + 1, kind=T.BF16), "aligned"), (dict(kind=5), "values"),
    (dict(slots=None), "null"), (dict(slots=P + 4), "aligned"), (dict(given=129), "128"), (dict(top=129), "128"), (dict(mask=P + 4), "aligned"), (dict(t=P + 2), "aligned"), (dict(lp=None), "null"),
    (dict(entropy=None), "null"), (dict(top_slots=None), "null"), (dict(top_lp=None), "null"), (dict(top_slots=P + 4), "aligned"), (dict(stats=P + 8), "aligned")])
def test_log_probs_refuses(change, text):
    refused(log_probs(**change), text)


@pytest.mark.parametrize("rows,n,top", [(1, 1_000_000, 0), (3, 10_000_000, 128)])
def test_log_probs_refuses_a_workspace_that_is_too_small(rows, n, top):
    need = T.lib().tv_log_probs_workspace(rows, n, top)
    if need == 0:
        pytest.skip("a call of this size needs none")
    refused(log_probs(rows=rows, n=n, top=top, ws_bytes=need - 1), "workspace")
    refused(log_probs(rows=rows, n=n, top=top, ws=None), "workspace")
    refused(log_probs(rows=rows, n=n, top=top, ws=P + 8), "workspace")


@pytest.mark.parametrize("change,text", [
    (dict(n=0), "without scores"), (dict(scores=None), "null"), (dict(kind=-1), "values"), (dict(slots=None), "null"), (dict(given=129), "128"), (dict(stats=None), "null"), (dict(stats=P + 4), "aligned"),
    (dict(g=P + 2), "aligned"), (dict(ge=P + 2), "aligned"), (dict(out=None), "null"), (dict(out=P + 2), "aligned"), (dict(out_stride=99), "overlap"), (dict(t=P + 1), "aligned"), (dict(mask=P + 1), "aligned")])
def test_log_probs_grad_refuses(change, text):
    refused(log_probs_grad(**change), text)


def test_no_rows_do_nothing():
    """Before any look at a device or a pointer that such a call does not need."""
    assert quantize(rows=0, x=None, codes=None, scales=None) == T.OK
    assert values(rows=0, codes=None, scales=None, out=None) == T.OK
    assert matmul(m=0, a=None, a_scales=None, out=None) == T.OK
    assert matmul(n=0, b=None, b_scales=None, out=None) == T.OK
    assert rms_norm(rows=0, x=None, codes=None, scales=None) == T.OK
    assert log_probs(rows=0, scores=None, slots=None, lp=None, entropy=None) == T.OK
    assert log_probs_grad(rows=0, scores=None, stats=None, out=None) == T.OK
    assert T.lib().tv_log_probs_workspace(0, 1 << 20, 128) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a call says where there is no GPU")
def test_no_device():
    for rc in (quantize(), values(), matmul(), rms_norm(), rms_norm(kind=T.ROWS_FP4, scale=T.SCALE_E8M0), log_probs(), log_probs_grad(), quantize(device=-1)):
        assert rc == T.ERR_NO_DEVICE


def test_python_refuses_before_the_library():
    x = torch.zeros(3, 256)
    codes, scales = torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(3, 8, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    rows8 = x.to(torch.float8_e4m3fn)
    for call, kind, text in (
            (lambda: fp4.quantize(x), ValueError, "on a GPU"),
            (lambda: fp4.quantize(x.numpy()), TypeError, "x must be a 2-D"),
            (lambda: fp4.quantize(x.double()), TypeError, "x must be a 2-D"),
            (lambda: fp4.Fp4Rows(codes, scales), ValueError, "on a GPU"),
            (lambda: fp4.Fp4Rows(x, scales), TypeError, "codes"),
            (lambda: fp4.matmul(codes, codes), TypeError, "Fp4Rows"),
            (lambda: fp4.matmul(rows8, codes), TypeError, "Fp4Rows"),
            (lambda: norm.rms_norm(x), ValueError, "on a GPU"),
            (lambda: norm.rms_norm(x[0]), TypeError, "x must be a 2-D"),
            (lambda: norm.add_rms_norm(x, None), TypeError, "residual"),
            (lambda: norm.add_rms_norm(x, x), ValueError, "on a GPU"),
            (lambda: sampling.log_probs(x, torch.zeros(3, dtype=torch.int64)), ValueError, "on a GPU"),
            (lambda: sampling.log_probs(x.long(), torch.zeros(3, dtype=torch.int64)), TypeError, "scores")):
        with pytest.raises(kind, match=text):
            call()
    assert fp8.BLOCK == 128 and fp4.BLOCK == 32
