"""Calls of the 8-bit floating-point operators that are refused by name, whatever is wrong with them, and values that are held
to the last bit."""
import pytest
import torch

from .test_gpu_fp8 import ACTS, F16, L, normal, weights  # noqa: F401
from .test_gpu_fp8_sums import check_rows

pytestmark = pytest.mark.gpu


def refused(L, name, call):
    with pytest.raises(L.LloomHipError) as e:
        call()
    assert e.value.name == name, str(e.value)


def test_starts_that_are_no_tensor(L):
    w, ws = (t.cuda() for t in weights(1, 3, 200, 256))
    x = torch.zeros(5, 256, device="cuda")
    for starts in (None, [0, 1, 2, 5], 0):
        refused(L, "EINVAL", lambda: L.fp8_grouped_matmul(x, w, ws, starts))
    starts = torch.tensor([0, 1, 2, 5], dtype=torch.int32, device="cuda")
    refused(L, "EINVAL", lambda: L.fp8_grouped_matmul(x, w, ws, starts, gather=[0, 1, 2, 3, 4]))
    refused(L, "EINVAL", lambda: L.fp8_grouped_matmul(x, w, ws, starts, scatter=[0, 1, 2, 3, 4]))


def test_more_experts_than_there_may_be(L):
    """Refused by their number, before memory for so many starts is asked for."""
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    free = torch.cuda.memory_reserved()
    for experts in (4097, 1 << 34, 1 << 45):
        refused(L, "ESHAPE", lambda: L.expert_plan(ids, experts))
    refused(L, "EINVAL", lambda: L.expert_plan(ids, -(1 << 45)))
    assert torch.cuda.memory_reserved() - free <= 2 << 20
    assert L.expert_plan(ids, 4096).starts.shape == (4097,)


@pytest.mark.parametrize("m", [3, 40, 700])
def test_outputs_that_share_memory_with_inputs(L, m):
    """Refused; side by side in one allocation they are served."""
    w, ws = (t.cuda() for t in weights(2, 256, 256))
    x = normal(m, m, 256, dtype=F16).cuda()
    want = L.fp8_matmul(x, w, ws)
    kept = x.clone()
    refused(L, "EINVAL", lambda: L.fp8_matmul(x, w, ws, out=x))
    both = torch.empty(2 * m + 1, 256, dtype=F16, device="cuda")
    both[:m] = x
    refused(L, "EINVAL", lambda: L.fp8_matmul(both[:m], w, ws, out=both[m - 1:2 * m - 1]))
    assert torch.equal(x, kept) and torch.equal(both[:m], kept)
    assert torch.equal(L.fp8_matmul(both[:m], w, ws, out=both[m:2 * m]), want)
    starts = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    refused(L, "EINVAL", lambda: L.fp8_grouped_matmul(x, w[None], ws[None], starts, out=x))
    want = L.fp8_grouped_matmul(x, w[None], ws[None], starts)  # may be served by another kernel: sums in another order
    assert torch.equal(L.fp8_grouped_matmul(both[:m], w[None], ws[None], starts, out=both[m:2 * m]), want)
    if m > 128:
        refused(L, "EINVAL", lambda: L.fp8_matmul(x[:128], w, ws, out=w.view(torch.uint8).view(F16).view(128, 256)))


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (5, 3, 144), (40, 7, 272), (600000, 1, 16), (200000, 3, 48), (90000, 7, 144)])
def test_few_columns(L, m, n, k, out):
    """Rows of y that begin at any place, by the kernel of few rows and by tiles."""
    w, ws = weights(n + k, n, k)
    q, sx = L.fp8_quantize(normal(m, m, k).cuda())
    y = L.fp8_matmul(q, w.cuda(), ws.cuda(), x_scales=sx, out_dtype=out)
    i = torch.unique(torch.cat([torch.arange(min(m, 40)), torch.arange(max(m - 40, 0), m)]))
    check_rows(y, q.cpu(), sx, w, ws, i)


@pytest.mark.parametrize("rows,n", [(3, 48), (50, 264), (900, 700)])
@pytest.mark.parametrize("act", ACTS)
def test_rows_gathered_from_none(L, rows, n, act):
    """x of no rows: every gather is out of range, so y is zeros, and it is reported."""
    w, ws = (t.cuda() for t in weights(2, 3, n, 272))
    starts = torch.tensor([0, rows // 2, rows // 2, rows], dtype=torch.int32, device="cuda")
    gather = torch.zeros(rows, dtype=torch.int32, device="cuda")
    y = L.fp8_grouped_matmul(torch.empty(0, 272, dtype=act, device="cuda"), w, ws, starts, gather=gather)
    assert y.shape == (rows, n) and not y.any()
    refused(L, "EEXPERT", L.paged_check)
    L.paged_check()


@pytest.mark.parametrize("dtype", ACTS)
@pytest.mark.parametrize("std", [0.01, 1.0, 4.0, 40.0])
def test_gate_has_the_bits_of_the_formula(L, std, dtype):
    """silu(gate) * up by the formula's four f32 operations, each rounded as IEEE says, and then rows into 8 bits: the same bytes
    and scales, everywhere, also where the exponential ends."""
    gate, up = normal(8, 1500, 2064, std=std).to(dtype), normal(9, 1500, 2064).to(dtype)
    gate[0] = torch.linspace(-130, 130, 2064)
    gate[1] = torch.linspace(-90, -79, 2064)
    gate[2, ::2], up[2, 1::2] = 0.0, 0.0
    gate[3, 5], gate[3, 500], up[3, 1000], up[4, 7] = float("nan"), float("-inf"), float("inf"), float("nan")
    g, u = gate.cuda(), up.cuda()
    q, s = L.fp8_silu_mul(g, u)
    q2, s2 = L.fp8_quantize(g.float() / (1.0 + torch.exp(-g.float())) * u.float())
    assert torch.equal(s, s2)
    a, b = q.view(torch.uint8), q2.view(torch.uint8)
    nan = (b & 127) == 127
    assert torch.equal((a & 127) == 127, nan) and torch.equal(a[~nan], b[~nan])
