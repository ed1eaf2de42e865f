"""The 8-bit floating-point operators where calls go wrong: refusals and reports, layouts, values that are no numbers, streams,
captures that are replayed, and a layer of experts with all of them together (bounds as in test_gpu_fp8.py)."""
import os
import sys

import numpy as np
import pytest
import torch

from . import fp8_ref as R
from .test_gpu_fp8 import ACTS, BF16, F16, F32, L, check_product, f64, normal, ragged, weights  # noqa: F401

pytestmark = pytest.mark.gpu


def expert_error(L):
    with pytest.raises(L.LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EEXPERT"
    L.paged_check()


# ------------------------------------------------------------- refusals --

def test_tensors_that_do_not_fit(L):
    w, ws = (t.cuda() for t in weights(1, 3, 200, 256))
    x, q = torch.zeros(5, 256, device="cuda"), torch.zeros(5, 256, device="cuda").to(torch.float8_e4m3fn)
    xs, starts = torch.ones(5, 2, device="cuda"), torch.tensor([0, 1, 2, 5], dtype=torch.int32, device="cuda")
    one, ones = w[0], ws[0]
    bad = [
        (2, lambda: L.fp8_quantize(x.long())), (2, lambda: L.fp8_quantize(q)), (3, lambda: L.fp8_quantize(x[:, :40])),
        (3, lambda: L.fp8_quantize(torch.zeros((), device="cuda"))), (3, lambda: L.fp8_silu_mul(x, x[:4])),
        (3, lambda: L.fp8_silu_mul(x, x.half())), (3, lambda: L.fp8_quantize_weight(x[0])),
        (2, lambda: L.fp8_quantize_weight(q)), (2, lambda: L.fp8_matmul(x.double(), one, ones)),
        (2, lambda: L.fp8_matmul(q, one, ones)), (2, lambda: L.fp8_matmul(x, one, ones, x_scales=xs)),
        (3, lambda: L.fp8_matmul(x[:, :128], one, ones)), (3, lambda: L.fp8_matmul(x, w, ws)),
        (3, lambda: L.fp8_matmul(x, one, ones[:1])), (3, lambda: L.fp8_matmul(x, one, ones[:, :1])),
        (3, lambda: L.fp8_matmul(x, w[:, :100].transpose(0, 1)[0], ones)), (2, lambda: L.fp8_matmul(x, one.float(), ones)),
        (2, lambda: L.fp8_matmul(x, one, ones.half())), (3, lambda: L.fp8_matmul(q, one, ones, x_scales=xs[:4])),
        (3, lambda: L.fp8_matmul(q, one, ones, x_scales=xs.half())), (2, lambda: L.fp8_matmul(x, one, ones, out_dtype=torch.float64)),
        (3, lambda: L.fp8_matmul(x, one, ones, out=torch.empty(5, 199, device="cuda"))),
        (3, lambda: L.fp8_matmul(x, one, ones, out=torch.empty(5, 200, device="cuda", dtype=F16))),
        (3, lambda: L.fp8_matmul(x, one, ones, out=torch.empty(200, 5, device="cuda").t())),
        (1, lambda: L.fp8_matmul(x, one, ones, out=torch.empty(1001, device="cuda")[1:].view(5, 200))),
        (3, lambda: L.fp8_matmul(x.cpu(), one, ones)), (2, lambda: L.expert_plan(x, 4)),
        (1, lambda: L.expert_plan(starts[:, None], 0)), (3, lambda: L.expert_plan(starts[:, None], 5000)),
        (3, lambda: L.fp8_grouped_matmul(x, w, ws, starts[:3])), (2, lambda: L.fp8_grouped_matmul(x, w, ws, starts.long())),
        (2, lambda: L.fp8_grouped_matmul(x, w, ws, starts, gather=starts.long())),
        (2, lambda: L.fp8_grouped_matmul(x, w, ws, starts, gather=starts.cpu())),
        (3, lambda: L.fp8_grouped_matmul(x, w, ws, starts, gather=starts, scatter=starts[:2])),
        (3, lambda: L.fp8_grouped_matmul(x[:3], w, ws, starts, scatter=starts)),
        (3, lambda: L.fp8_grouped_matmul(x, one, ones, starts)), (3, lambda: L.fp8_grouped_matmul(x, w, ws[:2], starts)),
        (3, lambda: L.fp8_grouped_matmul(x, w, ws, starts, out=torch.empty(4, 200, device="cuda"))),
    ]
    for i, (code, call) in enumerate(bad):
        with pytest.raises(L.LloomHipError) as e:
            call()
        assert e.value.code == code, (i, str(e.value))
    L.paged_check()  # nothing was launched that could report


# ---------------------------------------------------------- device reports --

@pytest.mark.parametrize("rows,n", [(7, 48), (40, 200), (900, 264)])
@pytest.mark.parametrize("starts", [[1, 2, 3, 7], [0, 5, 3, 7], [0, -1, 3, 7], [0, 2, 1 << 30, 1 << 30], [0, 2, 5, 100000],
                                    [-2 ** 31, 2 ** 31 - 1, 0, 3]])
def test_starts_out_of_order_leave_the_call_out(L, rows, n, starts):
    w, ws = weights(2, 3, n, 272)
    x = normal(3, rows, 272, dtype=F16)
    y = L.fp8_grouped_matmul(x.cuda(), w.cuda(), ws.cuda(), torch.tensor(starts, dtype=torch.int32).cuda())
    expert_error(L)
    assert y.shape == (rows, n) and not y.any()


@pytest.mark.parametrize("counts", [[3, 0, 4], [20, 31, 12], [300, 0, 400]])
def test_rows_out_of_range_are_left_out(L, counts):
    starts, rows, order = ragged(counts, 2, 4)
    w, ws = weights(5, 3, 136, 144)
    x = normal(6, 50, 144, dtype=BF16)
    gather, scatter = (order % 50).int(), order.int()
    lost_in, lost_out = [0, rows // 2], [1, rows // 3]
    gather[lost_in] = torch.tensor([50, -1], dtype=torch.int32)
    scatter[lost_out] = torch.tensor([rows, -7], dtype=torch.int32)
    out = torch.full((rows, 136), 7.0, dtype=BF16, device="cuda")
    y = L.fp8_grouped_matmul(x.cuda(), w.cuda(), ws.cuda(), starts.cuda(), gather=gather.cuda(), scatter=scatter.cuda(), out=out)
    expert_error(L)
    assert y is out
    y = y.cpu()
    for e, c in enumerate(counts):
        for i in range(int(starts[e]), int(starts[e]) + c):
            if i in lost_out:
                continue
            if i in lost_in:
                assert not y[scatter[i]].any()
            else:
                check_product(y[scatter[i]][None], x[gather[i]][None], None, w[e], ws[e])
    for i in lost_out:  # nothing went to the places that nothing names
        assert torch.all(y[order[i]] == 7.0)


def test_scatter_into_more_rows_leaves_the_others(L):
    counts = [5, 40, 3]
    starts, rows, _ = ragged(counts, 0, 1)
    w, ws = weights(6, 3, 72, 128)
    x = normal(7, rows, 128)
    place = torch.randperm(100, generator=torch.Generator().manual_seed(2))[:rows].int()
    out = torch.full((100, 72), -3.0, device="cuda")
    L.fp8_grouped_matmul(x.cuda(), w.cuda(), ws.cuda(), starts.cuda(), scatter=place.cuda(), out=out)
    L.paged_check()
    others = torch.ones(100, dtype=torch.bool)
    others[place.long()] = False
    out = out.cpu()
    assert torch.all(out[others] == -3.0)
    for e, c in enumerate(counts):
        i = slice(int(starts[e]), int(starts[e]) + c)
        check_product(out[place[i].long()], x[i], None, w[e], ws[e])


# ------------------------------------------------------------------ layouts --

@pytest.mark.parametrize("m", [1, 3, 16, 30, 70, 400])
def test_layouts_of_x(L, m):
    w, ws = weights(8, 264, 272)
    base = normal(m, m, 4 * 272, dtype=F16).cuda()
    for x in (base[:, 272:544], base[:, 8:280], base.view(2 * m, 544)[::2, :272], base[:, 4:276], base.view(m, 272, 4)[:, :, 1]):
        check_product(L.fp8_matmul(x, w.cuda(), ws.cuda()), x, None, w, ws)
    x = base.view(m, 2, 2, 272).transpose(1, 2)
    y = L.fp8_matmul(x, w.cuda(), ws.cuda(), out_dtype=F32)
    assert y.shape == (m, 2, 2, 264)
    check_product(y, x.contiguous(), None, w, ws)
    q, s = L.fp8_quantize(base[:, :544])
    wide = torch.rand(m, 15, device="cuda")  # scales of any strides
    part = wide[:, 1:13:2][:, :3]
    y = L.fp8_matmul(q[:, 272:], w.cuda(), ws.cuda(), x_scales=part)
    assert y.dtype is F32
    check_product(y, q[:, 272:], part, w, ws)


def test_out_and_default_types(L):
    w, ws = (t.cuda() for t in weights(9, 40, 64))
    x = normal(1, 6, 64, dtype=BF16).cuda()
    q, s = L.fp8_quantize(x)
    out = torch.empty(6, 40, dtype=F16, device="cuda")
    assert L.fp8_matmul(x, w, ws).dtype is BF16 and L.fp8_matmul(q, w, ws, x_scales=s).dtype is F32
    assert L.fp8_matmul(q, w, ws, x_scales=s, out=out) is out
    a = out.clone()
    assert torch.equal(L.fp8_matmul(q, w, ws, x_scales=s, out_dtype=F16), a)
    # both ways to 8 bits are one
    assert torch.equal(L.fp8_matmul(x, w, ws), L.fp8_matmul(q, w, ws, x_scales=s, out_dtype=BF16))


@pytest.mark.parametrize("out", ACTS)
def test_values_that_are_no_numbers_stay_in_their_row(L, out):
    for m, n in ((4, 96), (40, 96), (300, 1100), (2100, 300)):
        w, ws = weights(m, n, 400)
        x = normal(m + 1, m, 400, dtype=out)
        clean = L.fp8_matmul(x.cuda(), w.cuda(), ws.cuda())
        x[1, 5], x[m - 1, 399] = float("nan"), float("inf")
        wb = w.clone()
        wb.view(torch.uint8)[n - 1, 17] = 0x7F
        y = L.fp8_matmul(x.cuda(), wb.cuda(), ws.cuda())
        lost = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        lost[1] = lost[m - 1] = True
        lost[:, n - 1] = True
        assert torch.equal(y.isnan(), lost) and torch.equal(y[~lost], clean[~lost])


def test_scales_at_the_ends_of_their_range(L):
    """Rows and weights of huge and tiny scales whose products are ordinary numbers."""
    w, ws = weights(11, 64, 256)
    x = normal(12, 20, 256)
    q, s = (t.cpu() for t in L.fp8_quantize(x.cuda()))
    big, small = s * 2.0 ** 100, ws * 2.0 ** -100
    y = L.fp8_matmul(q.cuda(), w.cuda(), small.cuda(), x_scales=big.cuda())
    assert torch.equal(y, L.fp8_matmul(q.cuda(), w.cuda(), ws.cuda(), x_scales=s.cuda()))
    zero = L.fp8_matmul(torch.zeros(3, 256, device="cuda"), w.cuda(), ws.cuda())
    assert not zero.any()


def test_offsets_past_32_bits(L):
    """Weights of over 4 GB, rows of x of over 2 GB that are not gathered, and results of over 4 GB."""
    E, n, k = 9, 16384, 32768
    w = torch.zeros(E, n, k, dtype=torch.uint8, device="cuda")
    w[:, :, ::512] = torch.randint(0, 0x60, (E, n, k // 512), dtype=torch.uint8, device="cuda")
    w = w.view(torch.float8_e4m3fn)
    ws = torch.rand(E, n // 128, k // 128, device="cuda")
    starts = torch.tensor([0, 0, 1, 1, 1, 1, 1, 20, 20, 23], dtype=torch.int32, device="cuda")
    x = torch.randn(23, k, device="cuda")
    y = L.fp8_grouped_matmul(x, w, ws, starts)
    for e, i in ((1, 0), (6, 19), (8, 22)):
        want = L.fp8_matmul(x[i:i + 1], w[e], ws[e])
        assert (y[i] - want[0]).abs().max() <= 2.0 ** -18 * want.abs().max()
    del w, ws, y, x
    m, n, k = 140000, 16384, 16384 + 16
    q = torch.randint(0, 0x60, (m, k), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.rand(m, -(-k // 128), device="cuda")
    w, ws = (t.cuda() for t in weights(3, n, k))
    y = L.fp8_matmul(q, w, ws, x_scales=s, out_dtype=BF16)
    for i in (0, 70001, 131073, m - 1):
        want = L.fp8_matmul(q[i:i + 1], w, ws, x_scales=s[i:i + 1], out_dtype=F32)[0]
        # halves of a step, and what groups of eight products lose of a row's size
        assert (y[i].float() - want).abs().max() <= 2.0 ** -7 * want.abs().max()


# ---------------------------------------------------- streams and captures --

def test_another_stream(L):
    w, ws = (t.cuda() for t in weights(13, 520, 1024))
    x = normal(14, 300, 1024, dtype=F16).cuda()
    want = L.fp8_matmul(x, w, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        later = torch.zeros_like(x)
        for _ in range(20):
            later.add_(x)
        later.mul_(0).add_(x)
        got = L.fp8_matmul(later, w, ws)
        q, s = L.fp8_quantize(later)
    side.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(L.fp8_matmul(q, w, ws, x_scales=s, out_dtype=F16), want)


def layer(L, x, ids, up, down, experts):
    plan = L.expert_plan(ids, experts)
    h = L.fp8_grouped_matmul(x, *up, plan.starts, gather=plan.tokens)
    inner = h.shape[1] // 2
    q, s = L.fp8_silu_mul(h[:, :inner], h[:, inner:])
    return L.fp8_grouped_matmul(q, *down, plan.starts, x_scales=s, scatter=plan.planes, out_dtype=x.dtype)


@pytest.mark.parametrize("tokens,dtype", [(1, F16), (9, BF16), (200, F32), (700, F16)])
def test_a_layer_captured_and_replayed(L, tokens, dtype):
    E, topk, k, inner = 6, 2, 256, 144
    up = [t.cuda() for t in weights(15, E, 2 * inner, k)]
    down = [t.cuda() for t in weights(16, E, k, inner)]
    g = torch.Generator().manual_seed(tokens)

    def inputs():
        ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(tokens)]).int()
        if tokens > 4:
            ids[-2:] = -1
        return normal(int(torch.randint(1000, (), generator=g)), tokens, k, dtype=dtype).cuda(), ids.cuda()

    x, ids = (t.clone() for t in inputs())
    L.quantized.reserve_workspace(L.fp8_workspace_bytes(dtype, tokens * topk, k, x_rows=tokens, experts=E))
    layer(L, x, ids, up, down, E)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(L, x, ids, up, down, E)
    for _ in range(4):
        nx, ni = inputs()
        x.copy_(nx)
        ids.copy_(ni)
        graph.replay()
        got = y.clone()
        want = layer(L, nx, ni, up, down, E)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        # rows of padded tokens are zero
        if tokens > 4:
            assert not got[-2 * topk:].any()
    L.paged_check()


def test_a_capture_that_would_grow_the_workspace_is_refused(L):
    import ctypes

    from lloom_amd.lib import lib

    w, ws = (t.cuda() for t in weights(17, 264, 512))
    x, y = torch.zeros(4096, 512, device="cuda"), torch.zeros(4096, 264, device="cuda")
    ctx = ctypes.c_void_p()
    assert lib().lloom_hip_ctx_create(0, ctypes.byref(ctx)) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = lib().lloom_hip_fp8_matmul(ctx, w.data_ptr(), ws.data_ptr(), 264, 512, x.data_ptr(), 0, 512, None, 0, 0, 4096,
                                        y.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
        y.add_(1.0)
    assert rc == 6 and b"reserve" in lib().lloom_hip_last_error()
    graph.replay()
    assert torch.all(y == 1.0)
    del graph
    lib().lloom_hip_ctx_destroy(ctx)


# ----------------------------------------------------------------- together --

def exact_layer(x, ids, up, down):
    """The layer in 64 bits but for what its definition rounds: h to x's type and what goes through 8 bits."""
    E, inner = up[0].shape[0], up[0].shape[1] // 2
    y = np.zeros((ids.shape[0] * ids.shape[1], down[0].shape[1]))
    for p, e in enumerate(ids.reshape(-1).tolist()):
        if e < 0 or e >= E:
            continue
        q, sx = R.quantize(f64(x[p // ids.shape[1]])[None])
        h, _ = R.product(R.TABLE[q], sx, R.values(up[0][e]), f64(up[1][e]), F32, False)
        h = torch.from_numpy(h).to(x.dtype).double().numpy()
        a = h[:, :inner] / (1 + np.exp(-h[:, :inner])) * h[:, inner:]
        q, sx = R.quantize(a)
        y[p] = R.product(R.TABLE[q], sx, R.values(down[0][e]), f64(down[1][e]), F32, False)[0]
    return y


@pytest.mark.parametrize("tokens,dtype", [(1, BF16), (12, F32), (300, F16)])
def test_a_layer_of_experts(L, tokens, dtype):
    """Roundings of h that fall on the other side move what 8 bits make of it by a step (2^-4 of a value, in few places), so
    the layer is held to 2^-6 of the result's size in the 2-norm; with f32 no more than a few values can differ."""
    E, topk, k, inner = 5, 3, 192, 160
    up, down = weights(18, E, 2 * inner, k), weights(19, E, k, inner)
    g = torch.Generator().manual_seed(tokens)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(tokens)]).int()
    x = normal(20, tokens, k, dtype=dtype)
    y = layer(L, x.cuda(), ids.cuda(), [t.cuda() for t in up], [t.cuda() for t in down], E)
    assert y.dtype is dtype and y.shape == (tokens * topk, k)
    want = exact_layer(x, ids, up, down)
    assert np.linalg.norm(f64(y) - want) <= 2.0 ** -6 * np.linalg.norm(want)
    if dtype is F32:
        assert np.median(np.abs(f64(y) - want)) <= 1e-5 * np.abs(want).max()


def test_the_example(L):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import expert_layer

    worst, us = expert_layer.run(tokens=(1, 5, 130), steps=3)
    # A value m 2^e, 1 <= m < 2, is off by up to 2^-4 2^e evenly, 2^-4 / sqrt(3) = .036 in the square mean, and with 1 / m^2 on
    # average 3 / (8 ln 2) = .54 that is .0266 of itself.  x and the weight's make .0376 of g and u; of silu(g) u, whose
    # derivative by ln g is 1 + g (1 - sigmoid(g)) times it, 1.3 for g of 1, .0376 sqrt(1 + 1.3^2) = .062; with the 8 bits of
    # h and of the second weight sqrt(.062^2 + 2 * .0266^2) = .072 (the f32 products here have none of them).
    assert worst <= 0.1 and us > 0
