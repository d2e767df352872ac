"""Refusals of the operators beside the search, at the C ABI and in Python: no kernel is launched here and none would be."""
import ctypes as C

import pytest
import torch

from turbovec_amd import _lib as T
from turbovec_amd import fp8, sampling

P = 4096                       # a place that is never read


def refused(rc, text):
    assert rc == T.ERR_BAD_ARGUMENT and text in T.lib().tv_last_error().decode(), T.lib().tv_last_error()


def quantize(device=0, x=P, x_type=T.F32, x_stride=256, rows=4, dim=256, scale=T.SCALE_F32, group=1, codes=P, code_stride=256, scales=P, scale_stride=2):
    return T.lib().tv_fp8_quantize_dev(device, None, x, x_type, x_stride, rows, dim, scale, group, codes, code_stride, scales, scale_stride)


def matmul(m=4, n=4, dim=256, scale=T.SCALE_F32, group=1, a=P, a_scales=P, b=P, b_scales=P, out=P, out_type=T.F32, out_stride=4):
    return T.lib().tv_fp8_matmul_dev(0, None, a, dim, a_scales, 2, m, b, dim, b_scales, 2, n, group, dim, scale, out, out_type, out_stride)


def rescore(q=P, q_type=T.F32, nq=2, rows=P, scales=P, n=10, group=1, dim=256, scale=T.SCALE_F32, slots=P, m=8, k=4, s=P, i=P, ws=P, ws_bytes=1 << 20):
    return T.lib().tv_fp8_rescore_dev(0, None, q, q_type, dim, nq, rows, dim, scales, 2, n, group, dim, scale, slots, m, m, k, s, i, ws, ws_bytes)


def sample(scores=P, kind=T.F32, rows=2, n=100, mask=None, u=P, t=None, k=None, p=None, m=None, slots=P, probs=P, ws=P, ws_bytes=1 << 40):
    return T.lib().tv_sample_dev(0, None, scores, kind, n, rows, n, mask, 0, u, t, k, p, m, slots, probs, ws, ws_bytes)


@pytest.mark.parametrize("change,text", [
    (dict(dim=0), "dim"), (dict(dim=16385, code_stride=1 << 15), "dim"), (dict(rows=1 << 31), "too many rows"), (dict(scale=2), "scales"),
    (dict(group=64), "128"), (dict(group=0), "128"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(scales=P + 1), "aligned"),
    (dict(x_type=3), "values"), (dict(x=None), "null"), (dict(x=P + 2), "aligned"), (dict(code_stride=255), "overlap"), (dict(scale_stride=1), "overlap")])
def test_quantize_refuses(change, text):
    refused(quantize(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(dim=0), "dim"), (dict(m=1 << 31), "rows"), (dict(n=1 << 31), "rows"), (dict(scale=-1), "scales"), (dict(group=2), "128"), (dict(a=None), "null"),
    (dict(b=None), "null"), (dict(a_scales=None), "null"), (dict(b_scales=P + 2), "aligned"), (dict(out=None), "null"), (dict(out=P + 2), "aligned"),
    (dict(out_type=9), "values"), (dict(out_stride=3), "overlap")])
def test_matmul_refuses(change, text):
    refused(matmul(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(dim=20000), "dim"), (dict(k=9), "k exceeds"), (dict(m=16385, ws_bytes=1 << 30), "16384"), (dict(q=None), "null"), (dict(q=P + 2), "aligned"),
    (dict(slots=None), "null"), (dict(slots=P + 4), "aligned"), (dict(s=None), "null"), (dict(i=P + 4), "aligned"), (dict(ws=None, m=300), "workspace"),
    (dict(ws_bytes=2 * 300 * 8 - 1, m=300), "workspace"), (dict(ws=P + 4, m=300), "workspace"), (dict(rows=None), "null"), (dict(group=3), "128"), (dict(q_type=7), "values"), (dict(nq=1 << 31, ws_bytes=1 << 40), "queries")])
def test_rescore_refuses(change, text):
    refused(rescore(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(n=0), "without scores"), (dict(n=1 << 31), "too many"), (dict(rows=1 << 31), "too many"), (dict(scores=None), "null"), (dict(scores=P + 1, kind=T.BF16), "aligned"),
    (dict(u=None), "null"), (dict(slots=None), "null"), (dict(probs=None), "null"), (dict(t=P + 2), "aligned"), (dict(mask=P + 4), "aligned"), (dict(kind=5), "values")])
def test_sample_refuses(change, text):
    refused(sample(**change), text)


def test_no_rows_do_nothing():
    """Before any look at a device or a pointer that such a call does not need."""
    assert quantize(rows=0, x=None, codes=None, scales=None) == T.OK
    assert matmul(m=0, a=None, a_scales=None, out=None) == T.OK
    assert matmul(n=0, b=None, b_scales=None, out=None) == T.OK
    assert rescore(nq=0, ws=None, ws_bytes=0) == T.OK
    assert rescore(k=0) == T.OK
    assert rescore(m=0, k=0, slots=None) == T.OK
    assert sample(rows=0, scores=None) == T.OK
    assert T.lib().tv_sample_workspace(0, 1 << 20) == 0 and T.lib().tv_fp8_rescore_workspace(0, 1000, 256) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a call says where there is no GPU")
def test_no_device():
    for rc in (quantize(), matmul(), rescore(), sample()):
        assert rc == T.ERR_NO_DEVICE
    n = C.c_int(0)
    assert quantize(device=-1) == T.ERR_NO_DEVICE, n


def test_python_refuses_before_the_library():
    x = torch.zeros(3, 256)
    codes, scales = torch.zeros(3, 256).to(torch.float8_e4m3fn), torch.zeros(3, 2)
    for call, kind, text in (
            (lambda: fp8.quantize(x), ValueError, "on a GPU"),
            (lambda: fp8.quantize(x.numpy()), TypeError, "x must be a 2-D"),
            (lambda: fp8.quantize(x.double()), TypeError, "x must be a 2-D"),
            (lambda: fp8.quantize(x[0]), TypeError, "1-D"),
            (lambda: fp8.Fp8Rows(codes, scales), ValueError, "on a GPU"),
            (lambda: fp8.Fp8Rows(x, scales), TypeError, "codes"),
            (lambda: fp8.matmul(codes, codes), TypeError, "Fp8Rows"),
            (lambda: fp8.rescore(x, codes, x.long(), 1), TypeError, "Fp8Rows"),
            (lambda: sampling.sample(x, torch.zeros(3)), ValueError, "on a GPU"),
            (lambda: sampling.sample(x.long(), torch.zeros(3)), TypeError, "scores")):
        with pytest.raises(kind, match=text):
            call()
