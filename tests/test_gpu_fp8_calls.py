"""Calls of the 8-bit floating-point operators that are refused by name, whatever is wrong with them, and values that are held
to the last bit."""
import pytest
import torch

from .test_gpu_fp8 import ACTS, F16, F32, L, check_product, normal, weights  # noqa: F401

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
