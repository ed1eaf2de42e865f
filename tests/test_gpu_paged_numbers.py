"""Attention over the paged cache where q, keys or values hold infinities or NaN: a row is what the definition makes of
what it sees, whether its keys are split among workgroups or not, and the other rows are left alone."""
import math

import pytest
import torch

import lloom_amd as L

from . import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, F32 = torch.float16, torch.float32

#            cached, new, page, kv_heads, group
WAYS = {
    "first_token": ([0], [1], 16, 2, 4), "few_rows": ([40, 300], [3, 1], 16, 2, 3),
    "few_rows_split": ([9, 30000], [1, 3], 64, 1, 4), "tiles": ([300, 5], [130, 1], 32, 1, 2),
    "tiles_split": ([6000], [90], 64, 1, 2), "many_requests": ([3 * i for i in range(70)], [1 + 60 * (i == 9) for i in range(70)], 16, 1, 2),
}


def _run(s, **kw):
    return L.paged_attention(s["q"], s["k"], s["v"], s["t_tables"], s["t_start"], s["t_lens"], **kw)


def _check(s, got, window=0, sinks=0):
    """got is the definition's: NaN in the same places, within the bound elsewhere.  Scores' bounds are those of the keys
    before any was spoilt (s["whole"])."""
    args = s["tables"], s["q_start"], s["seq_lens"], s["scale"], window, sinks
    want, mass, reach, count = R.attention(s["q"], s["k"], s["v"], *args)
    if "whole" in s:
        reach = R.attention(s["q"], s["whole"], s["v"], *args)[2]
    tol = R.bound(want, mass, reach, count, s["q"].dtype, s["q"].shape[-1])
    got = got.double().cpu()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    assert ((got - want).abs() <= tol)[~nan].all()
    return nan


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("way", WAYS)
def test_a_query_that_is_no_number(way, dim, bad, act):
    s = R.case(*WAYS[way], dim, act, device=DEV)
    spoilt = [(0, 1), (s["q"].shape[0] - 1, 0), (s["q"].shape[0] // 2, s["q"].shape[1] - 1)]
    for row, head in spoilt:
        s["q"][row, head, (row + 7 * head) % dim] = bad
    nan = _check(s, _run(s))
    assert all(nan[at].all() for at in spoilt) and int(nan.sum()) == len(set(spoilt)) * dim
    L.paged_check()


SPOILT = [(0, 1), (0, 150), (70, 75), (0, 10 ** 6)]


def _minus_infinity(way, first, last, act):
    """Keys first .. last - 1 of every request have scores of -inf."""
    s = R.case(*WAYS[way], 64, act, device=DEV)
    s["q"][..., 5] = s["q"][..., 5].abs() + 0.5
    page = s["k"].shape[2]
    s["whole"] = s["k"].clone()
    for b, length in enumerate(s["seq_lens"]):
        for p in range(first, min(last, length)):
            s["k"][s["tables"][b][p // page], :, p % page, 5] = -math.inf
    return s


@pytest.mark.parametrize("first,last", SPOILT)
@pytest.mark.parametrize("way", WAYS)
def test_keys_whose_scores_are_minus_infinity(way, first, last):
    """They get no weight; a row that sees no others has no softmax: NaN."""
    s = _minus_infinity(way, first, last, F16)
    nan = _check(s, _run(s))
    assert last < 10 ** 6 or nan.all()
    _check(s, _run(s, window=40), 40)
    _check(s, _run(s, window=40, sinks=3), 40, 3)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("first,last", [(0, 1), (70, 75), (20, 40)])
@pytest.mark.parametrize("way", WAYS)
def test_values_that_are_no_numbers_at_keys_of_no_weight(way, first, last, bad):
    """Zero times them is NaN, in the rows that see them, wherever the key is in a step that not all rows see whole."""
    s = _minus_infinity(way, first, last, F16)
    page = s["k"].shape[2]
    for b, length in enumerate(s["seq_lens"]):
        for p in range(first, min(last, length)):
            s["v"][s["tables"][b][p // page], :, ::3, p % page] = bad
    nan = _check(s, _run(s))
    assert nan[..., ::3].any() or max(s["seq_lens"]) <= first
    _check(s, _run(s, window=40), 40)
    _check(s, _run(s, window=40, sinks=3), 40, 3)


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("large", [2.0 ** 6, 2.0 ** 12, 2.0 ** 16])
def test_f32_queries_with_one_large_value(way, large):
    """The others keep their bits beside it.  (What is left of a value is under 2^-22 of it or, with the row's largest at
    2^14 or more, half of half's least step, 2^-25, which is 2^-39 of the largest: 2^-23 here, of values of size 2.4.
    The keys are zero where the large one is, so that the bound is that of the others.)"""
    s = R.case(*WAYS[way], 64, F32, device=DEV)
    s["q"] = s["q"] * 1.5
    s["q"][..., 9] = large
    s["k"][..., 9].mul_(0.0)
    _check(s, _run(s))


@pytest.mark.parametrize("first,last", SPOILT)
@pytest.mark.parametrize("way", WAYS)
def test_infinite_keys_and_f32_queries(way, first, last):
    """Scores of -inf as from f16 queries, also where a query's value is exact in one half, or is none."""
    s = _minus_infinity(way, first, last, F32)
    s["q"][::3, :, 5] = s["q"][::3, :, 5].half().float()
    s["q"][1::3, ::2, 5] = 0.25
    nan = _check(s, _run(s))
    assert last < 10 ** 6 or nan.all()
    _check(s, _run(s, window=40, sinks=3), 40, 3)
    s["q"][:, -1, 5] = 0.0  # zero times it is NaN
    nan = _check(s, _run(s))
    assert nan[:, -1].any() or max(s["seq_lens"]) <= first


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("weight", [0.5 + 2.0 ** -12 - 2.0 ** -18, 0.5 + 2.0 ** -12 + 2.0 ** -18, 0.75 + 2.0 ** -12 - 2.0 ** -17])
@pytest.mark.parametrize("cached,new", [(299, 1), (999, 3), (200, 100), (900, 90)])
def test_values_that_are_all_alike_come_out_as_they_are(cached, new, weight, act):
    """A key of weight 1 in 32, so that whoever sums a few of them has it, and others of `weight`, which half rounds by
    nearly half a step: a sum of weights that was not of those that the values are summed with would show that in full.  The result is off by the roundings of both sums, 2 n +
    64 of half an f32 step, and f32's weights by twice 2^-22: 1.3e-4 at 1002 keys, under the half step of 2^-12 to the
    number below 1 in f16, so that there it is 1, -1, 0.5 and 2 exactly."""
    s = R.case([cached], [new], 16, 1, 4, 64, act, device=DEV)
    s["k"].zero_(), s["q"].zero_()
    s["q"][..., 3] = 1.0
    s["k"][s["tables"][0][::2], :, 5, 3] = 1.0
    worth = torch.tensor([1.0, -1.0, 0.5, 2.0], device=DEV).repeat(16)
    s["v"][:] = worth[:, None]
    got = _run(s, scale=-math.log(weight))
    n = cached + new
    tol = 0.0 if act == F16 else ((2 * n + 64) * 2.0 ** -24 + 2 * 2.0 ** -22)
    assert ((got.double() - worth).abs() <= tol * worth.abs()).all()


@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e20, 3e37])
@pytest.mark.parametrize("way", WAYS)
def test_f32_queries_of_any_size(way, size):
    """q over f32's range, with a scale that makes of it scores of ordinary size."""
    s = R.case(*WAYS[way], 64, F32, device=DEV)
    q = s["q"]
    s["q"] = q * size
    s["scale"] = 0.125 / size
    _check(s, _run(s, scale=s["scale"]))
