"""The refusals of the 8-bit floating-point calls, which need no GPU (every call below is refused before anything is read), and
the plain implementations that their GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import lloom_amd as L
from lloom_amd.lib import LloomHipError, lib

from . import fp8_ref as R

PTR = 1 << 20  # a 16-byte aligned address that nothing reads
EINVAL, EDTYPE, ESHAPE = 1, 2, 3


def _quantize(**kw):
    a = dict(ctx=PTR, x=PTR, dtype=0, stride=256, rows=4, k=256, q=PTR, s=PTR, ss=4, stream=None)
    a.update(kw)
    return lib().lloom_hip_fp8_quantize(*a.values())


def _gate(**kw):
    a = dict(ctx=PTR, g=PTR, gs=256, u=PTR, us=256, dtype=1, rows=4, k=256, q=PTR, s=PTR, ss=4, stream=None)
    a.update(kw)
    return lib().lloom_hip_fp8_silu_mul(*a.values())


def _weight(**kw):
    a = dict(ctx=PTR, w=PTR, dtype=30, experts=2, n=100, k=256, q=PTR, s=PTR, stream=None)
    a.update(kw)
    return lib().lloom_hip_fp8_quantize_weight(*a.values())


def _matmul(**kw):
    a = dict(ctx=PTR, w=PTR, ws=PTR, n=100, k=256, x=PTR, dtype=100, stride=256, xs=PTR, xs_row=2, xs_block=1, m=4, y=PTR,
             out=0, stream=None)
    a.update(kw)
    return lib().lloom_hip_fp8_matmul(*a.values())


def _grouped(**kw):
    a = dict(ctx=PTR, w=PTR, ws=PTR, experts=4, n=100, k=256, x=PTR, dtype=100, stride=256, xs=PTR, xs_row=2, xs_block=1,
             x_rows=4, starts=PTR, gather=None, scatter=None, rows=4, y=PTR, out=0, y_rows=4, stream=None)
    a.update(kw)
    return lib().lloom_hip_fp8_grouped_matmul(*a.values())


def _plan(**kw):
    a = dict(ctx=PTR, ids=PTR, tokens=4, topk=2, experts=8, starts=PTR, planes=PTR, of=PTR, stream=None)
    a.update(kw)
    return lib().lloom_hip_expert_plan(*a.values())


def refused(call, kw, code, name):
    assert call(**kw) == code
    assert name in lib().lloom_hip_last_error()


ROWS = [(dict(ctx=None), EINVAL), (dict(q=None), EINVAL), (dict(s=None), EINVAL), (dict(dtype=12), EDTYPE),
        (dict(dtype=100), EDTYPE), (dict(k=0), EINVAL), (dict(k=-16), EINVAL), (dict(k=24), ESHAPE), (dict(k=1 << 23), ESHAPE),
        (dict(rows=-1), EINVAL), (dict(rows=(1 << 24) + 1, ss=1 << 25), ESHAPE), (dict(ss=3), ESHAPE), (dict(q=PTR + 4), EINVAL),
        (dict(s=PTR + 2), EINVAL), (dict(rows=1 << 24, ss=1 << 24, k=8192), ESHAPE)]


@pytest.mark.parametrize("kw,code", ROWS + [(dict(x=None), EINVAL), (dict(stride=255), ESHAPE), (dict(stride=258), EINVAL),
                                            (dict(x=PTR + 8), EINVAL)])
def test_quantize_refusals(kw, code):
    refused(_quantize, kw, code, b"fp8_quantize")


@pytest.mark.parametrize("kw,code", ROWS + [(dict(g=None), EINVAL), (dict(u=None), EINVAL), (dict(gs=128), ESHAPE),
                                            (dict(us=255), ESHAPE), (dict(us=260), EINVAL), (dict(u=PTR + 2), EINVAL)])
def test_gate_refusals(kw, code):
    refused(_gate, kw, code, b"fp8_silu_mul")


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), EINVAL), (dict(w=None), EINVAL), (dict(dtype=100), EDTYPE), (dict(k=100), ESHAPE), (dict(n=0), EINVAL),
    (dict(experts=0), EINVAL), (dict(experts=5000), ESHAPE), (dict(n=1 << 24, k=1 << 22), ESHAPE), (dict(w=PTR + 8), EINVAL),
    (dict(q=PTR + 4), EINVAL), (dict(s=PTR + 1), EINVAL)])
def test_weight_refusals(kw, code):
    refused(_weight, kw, code, b"fp8_quantize_weight")


PRODUCT = [(dict(ctx=None), EINVAL), (dict(w=None), EINVAL), (dict(ws=None), EINVAL), (dict(x=None), EINVAL),
           (dict(y=None), EINVAL), (dict(xs=None), EINVAL), (dict(dtype=8), EDTYPE), (dict(out=100), EDTYPE), (dict(out=8), EDTYPE),
           (dict(n=0), EINVAL), (dict(n=1 << 25), ESHAPE), (dict(k=0), EINVAL), (dict(k=250), ESHAPE), (dict(stride=128), ESHAPE),
           (dict(stride=264), EINVAL), (dict(dtype=1, stride=260), EINVAL), (dict(x=PTR + 8), EINVAL), (dict(w=PTR + 8), EINVAL),
           (dict(y=PTR + 8), EINVAL), (dict(xs=PTR + 2), EINVAL), (dict(xs_row=-1), EINVAL), (dict(xs_block=-1), EINVAL)]


@pytest.mark.parametrize("kw,code", PRODUCT + [
    (dict(m=-1), EINVAL), (dict(m=1 << 25), ESHAPE), (dict(m=1 << 24, n=1 << 24), ESHAPE),
    # a tile's rows, and the scales, within 32-bit offsets
    (dict(stride=1 << 23), ESHAPE), (dict(xs_row=1 << 21), ESHAPE), (dict(xs_block=1 << 29), ESHAPE)])
def test_matmul_refusals(kw, code):
    refused(_matmul, kw, code, b"fp8_matmul")


@pytest.mark.parametrize("kw,code", PRODUCT + [
    (dict(starts=None), EINVAL), (dict(rows=-1), EINVAL), (dict(y_rows=-1), EINVAL), (dict(x_rows=-1), EINVAL),
    (dict(experts=0), EINVAL), (dict(experts=4097), ESHAPE), (dict(x_rows=3), ESHAPE), (dict(y_rows=3), ESHAPE),
    (dict(rows=(1 << 24) + 1, x_rows=1 << 24, y_rows=1 << 24, gather=PTR), ESHAPE),
    # all rows that may be gathered within 32-bit offsets
    (dict(gather=PTR, x_rows=1 << 23), ESHAPE), (dict(gather=PTR, x_rows=1 << 20, xs_row=1 << 9), ESHAPE)])
def test_grouped_refusals(kw, code):
    refused(_grouped, kw, code, b"fp8_grouped_matmul")


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), EINVAL), (dict(ids=None), EINVAL), (dict(starts=None), EINVAL), (dict(planes=None), EINVAL),
    (dict(of=None), EINVAL), (dict(tokens=-1), EINVAL), (dict(topk=0), EINVAL), (dict(experts=0), EINVAL),
    (dict(experts=4097), ESHAPE), (dict(topk=4097), ESHAPE), (dict(tokens=1 << 23), ESHAPE), (dict(tokens=1 << 62, topk=4), ESHAPE)])
def test_plan_refusals(kw, code):
    refused(_plan, kw, code, b"expert_plan")


def test_workspace_bytes():
    ws = L.fp8_workspace_bytes
    assert ws(torch.float8_e4m3fn, 4096, 2048) == 0
    assert ws(torch.float16, 1, 2048) == 0  # brought into 8 bits where it is read
    assert 4096 * 2048 < ws(torch.bfloat16, 4096, 2048) <= 4096 * (2048 + 64) + 256
    assert ws(torch.float32, 65536, 2048, x_rows=8192, experts=64) <= 8192 * (2048 + 64) + 256
    out = ctypes.c_size_t()
    for args, code in (((12, 1, 1, 0, 256), EDTYPE), ((0, -1, 1, 0, 256), EINVAL), ((0, 1, 1, -1, 256), EINVAL),
                       ((0, 1, 1, 0, 100), ESHAPE), ((0, 1 << 25, 1, 0, 256), ESHAPE), ((0, 1, 1, 5000, 256), ESHAPE)):
        assert lib().lloom_hip_fp8_workspace_bytes(*args, ctypes.byref(out)) == code
    assert lib().lloom_hip_fp8_workspace_bytes(0, 1, 1, 0, 256, None) == EINVAL


def test_tensors_that_are_on_no_gpu_are_refused():
    x, w, s = torch.zeros(2, 32), torch.zeros(16, 32).to(torch.float8_e4m3fn), torch.ones(1, 1)
    for call in (lambda: L.fp8_quantize(x), lambda: L.fp8_silu_mul(x, x), lambda: L.fp8_quantize_weight(x),
                 lambda: L.fp8_matmul(x, w, s), lambda: L.expert_plan(torch.zeros(2, 2, dtype=torch.int32), 4),
                 lambda: L.fp8_grouped_matmul(x, w[None], s[None], torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(LloomHipError, match="HIP device"):
            call()


# the plain implementations against what e4m3 is known to be

def test_table():
    t = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.TABLE, t, equal_nan=True)


def test_nearest():
    v = torch.cat([torch.linspace(-448, 448, 20011), torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, -21.0])]).double()
    got = R.nearest(v.numpy())
    want = v.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    zero = R.TABLE[got] == 0
    assert np.array_equal(got[~zero], want[~zero]) and np.all(R.TABLE[want[zero]] == 0)


def test_scale():
    s = R.scale(np.array([0.0, 448.0, 449.0, 224.0, 224.5, 2.0 ** -130, 2.0 ** -117, 1e38]))
    assert s.tolist() == [1.0, 1.0, 2.0, 0.5, 1.0, 2.0 ** -126, 2.0 ** -125, 2.0 ** 118]
