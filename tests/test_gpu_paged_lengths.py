"""Attention over the paged cache where lengths, windows and first tokens are near the largest there are."""
import pytest
import torch

import lloom_amd as L
from lloom_amd.lib import LloomHipError

from . import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, F32 = torch.float16, torch.float32
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("length", [MOST, 2 ** 30, MOST - 200])
@pytest.mark.parametrize("window,sinks", [(0, 0), (10, MOST), (10, 2 ** 30), (10, 3), (10, 0), (MOST, 0), (MOST, MOST), (2 ** 30 + 7, 40)])
@pytest.mark.parametrize("new,blocks", [(1, 9), (90, 20), (1, 300)])
def test_lengths_far_past_the_table(new, blocks, window, sinks, length, act):
    """Every token is past all keys that the table has places for: it sees those that it would, and the call is reported.
    The reference has each token as a request of its own, at a position that sees the same keys."""
    page, have = 16, 16 * blocks
    s = R.case([have - 1], [1], page, 1, 2, 64, act, device=DEV)
    q = (2 * torch.randn(new, 2, 64, generator=torch.Generator().manual_seed(new))).to(act).to(DEV)
    got = L.paged_attention(q, s["k"], s["v"], s["t_tables"], torch.tensor([0, new], dtype=torch.int32, device=DEV),
                            torch.tensor([length], dtype=torch.int32, device=DEV), window=window, sinks=sinks)
    with pytest.raises(LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EPAGE"
    for i in range(new):
        p = length - new + i  # sees keys under `sinks`, or from `first` on
        first = max(0, p - window + 1) if window else 0
        assert first == 0 or first >= have
        seen = min(sinks, have) if first else have
        want, *rest = R.attention(q[i:i + 1], s["k"], s["v"], s["tables"], [0, 1], [seen], s["scale"], 0, 0)
        tol = R.bound(want, *rest, act, 64)
        assert ((got[i:i + 1].double().cpu() - want).abs() <= tol).all(), i
