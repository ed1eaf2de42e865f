"""Attention over the paged cache: which rows of q a request owns, where q_start is not simply 0 .. tokens."""
import pytest
import torch

import lloom_amd as L
from lloom_amd.lib import LloomHipError

from . import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, F32 = torch.float16, torch.float32

#            cached, new, page, kv_heads, group, dim
WAYS = {
    "few_rows": ([40, 0, 300], [3, 1, 1], 16, 2, 3, 64), "few_rows_split": ([9, 30000], [1, 3], 64, 1, 4, 64),
    "tiles": ([300, 5], [130, 1], 32, 1, 2, 128), "tiles_split": ([6000, 0], [90, 70], 64, 1, 2, 64),
    "many_requests": ([3 * i for i in range(70)], [1 + 60 * (i == 9) for i in range(70)], 16, 1, 2, 96),
}


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _run(s, **kw):
    out = torch.full_like(s["q"], 7.0)
    return L.paged_attention(s["q"], s["k"], s["v"], s["t_tables"], s["t_start"], s["t_lens"], out=out, **kw)


def _check(s, got):
    """got is the definition's within the bound, zero where no request owns the row."""
    want, *rest = R.attention(s["q"], s["k"], s["v"], s["tables"], s["q_start"], s["seq_lens"], s["scale"], 0, 0)
    tol = R.bound(want, *rest, s["q"].dtype, s["q"].shape[-1])
    assert ((got.double().cpu() - want).abs() <= tol).all()
    owned = torch.zeros(got.shape[0], dtype=torch.bool)
    owned[s["q_start"][0]:s["q_start"][-1]] = True
    assert (got[~owned] == 0).all()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("before,after", [(1, 0), (5, 3), (300, 0)])
@pytest.mark.parametrize("way", WAYS)
def test_rows_before_the_first_request(way, before, after, act):
    """A part of a longer step's starts, with all of its rows."""
    s = R.case(*WAYS[way], act, pad=before + after, device=DEV)
    s["q_start"] = [before + n for n in s["q_start"]]
    s["t_start"] = _ints(s["q_start"])
    _check(s, _run(s))
    _check(s, _run(s, max_new=max(WAYS[way][1])))
    L.paged_check()


def _reported():
    with pytest.raises(LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EPAGE"
    L.paged_check()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("way", WAYS)
def test_starts_that_fall_leave_the_call_out(way, act):
    """Zeros and a report, and the next call's splits are joined as ever."""
    s = R.case(*WAYS[way], act, device=DEV)
    want = _run(s)
    n, good = s["q"].shape[0], s["t_start"]
    for start in ([n, 0], [0, n, 0, n], [0, n - 1, n - 2, n], [-1, n], [-n, 0, n], [-2 ** 31, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31]):
        # the requests beyond: in place in the middle of the others, so that more than one wave's worth is looked at
        q_start = (start + [start[-1]] * len(s["seq_lens"]))[:len(s["seq_lens"]) + 1]
        if len(s["seq_lens"]) > 64:
            q_start = [0] * (len(s["seq_lens"]) + 1 - len(start)) + start
        if all(a <= b for a, b in zip(q_start, q_start[1:])) and q_start[0] >= 0:
            continue
        s["t_start"] = _ints(q_start)
        assert (_run(s) == 0).all(), q_start
        s["t_start"] = good
        assert torch.equal(_run(s), want), q_start
        _reported()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("cut", [1, 3, 64])
@pytest.mark.parametrize("way", WAYS)
def test_rows_that_are_not_there(way, cut, act):
    """q without the last rows of the step: the others are at the positions that they had, and the call is reported."""
    s = R.case(*WAYS[way], act, device=DEV)
    cut = min(cut, s["q"].shape[0] - 1)
    want, *rest = R.attention(s["q"], s["k"], s["v"], s["tables"], s["q_start"], s["seq_lens"], s["scale"], 0, 0)
    tol = R.bound(want, *rest, act, s["q"].shape[-1])
    _run(s)
    L.paged_check()
    s["q"] = s["q"][:-cut]
    got = _run(s)
    assert ((got.double().cpu() - want[:-cut]).abs() <= tol[:-cut]).all()
    _reported()
    # as a plan for fewer rows than there are new tokens says
    cached, new = WAYS[way][:2]
    plan = L.paged_plan(_ints(cached), _ints(new), s["q"].shape[0], s["t_tables"], _ints([0] * 4096), WAYS[way][2])
    assert plan.q_start.tolist() == s["q_start"] and plan.seq_lens.tolist() == s["seq_lens"]
    _reported()


@pytest.mark.parametrize("tables,free", [([[3, -1, 0], [5, 0, 0]], [7, 8]), ([[3, 4, 0], [5, 0, 0]], [7, -2]), ([[3, 4, 0], [-2 ** 31, 0, 0]], [7, 8])])
def test_a_plan_reports_pages_that_are_none(tables, free):
    """Tokens whose page is negative, in the table of what a request holds or in the free list."""
    cached, new = [20, 10], [14, 20]
    got = L.paged_plan(_ints(cached), _ints(new), 34, _ints(tables), _ints(free), 16)
    _reported()
    start, lens, pos, slots, taken, after = R.plan(cached, new, 34, tables, free, 16)
    assert got.slots.tolist() == slots and -1 in slots and got.positions.tolist() == pos
    assert got.q_start.tolist() == start and got.seq_lens.tolist() == lens and got.taken.tolist() == [taken]
    assert got.block_tables.tolist() == after
