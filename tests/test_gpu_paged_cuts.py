"""Attention over the paged cache, in every way a call is cut: tiles and splits whose keys are a window's and the first
tokens, calls of more requests than a wave has lanes (up to as many as a call may have), and what is no number among them."""
import math

import pytest
import torch

import lloom_amd as L

from . import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, F32 = torch.float16, torch.float32


def _run(s, **kw):
    out = torch.full_like(s["q"], 7.0)
    return L.paged_attention(s["q"], s["k"], s["v"], s["t_tables"], s["t_start"], s["t_lens"], out=out, **kw)


def _dense(s, b, window, sinks):
    """Request b from the definition in 64 bits on the GPU, and what R.bound takes."""
    first, end, length = s["q_start"][b], s["q_start"][b + 1], s["seq_lens"][b]
    key = torch.arange(length, device=DEV)
    pages, kv_heads, page, dim = s["k"].shape
    home = s["t_tables"][b].long()[key // page]
    pos = torch.arange(length - (end - first), length, device=DEV)[:, None]
    seen = key <= pos
    if window:
        seen &= (key > pos - window) | (key < sinks)
    q = s["q"][first:end].double()
    heads = q.shape[1]
    out, mass, reach = torch.empty_like(q), torch.empty_like(q), torch.empty(end - first, heads, device=DEV, dtype=torch.float64)
    for h in range(heads):
        j = h // (heads // kv_heads)
        k, v = s["k"][home, j, key % page].double(), s["v"][home, j, :, key % page].double()
        z = s["scale"] * torch.mm(q[:, h], k.t().contiguous())
        w = torch.softmax(z.masked_fill(~seen, -math.inf), 1)
        out[:, h], mass[:, h] = torch.mm(w, v), torch.mm(w, v.abs())
        far = s["scale"] * torch.mm(q[:, h].abs(), k.abs().t().contiguous())
        reach[:, h] = far.masked_fill(~seen, 0.0).amax(1)
    count = seen.sum(1, keepdim=True).float().expand(-1, heads)
    return out.cpu(), mass.cpu(), reach.cpu(), count.cpu()


def _check(s, window, sinks, *outs):
    outs = [o.double().cpu() for o in outs]
    for b in range(len(s["seq_lens"])):
        rows = slice(s["q_start"][b], s["q_start"][b + 1])
        if rows.start == rows.stop:
            continue
        want, *rest = _dense(s, b, window, sinks)
        tol = R.bound(want, *rest, s["q"].dtype, s["q"].shape[-1])
        for o in outs:
            assert ((o[rows] - want).abs() <= tol).all(), (b, ((o[rows] - want).abs() / tol).max())


#            cached, new, page, kv_heads, group, dim
SPLIT = {
    "one_chunk": ([6000], [512], 64, 4, 4, 64), "short_chunk": ([9000], [90], 16, 1, 2, 128), "few_rows": ([30000], [9], 16, 1, 4, 128),
    "rows_beside_tiles": ([30000, 20000, 25000, 9000], [1, 300, 2, 1], 32, 2, 4, 64),
    "wide_heads": ([9000, 5000], [70, 1], 32, 1, 2, 256), "heads_of_96": ([7000, 40], [200, 33], 128, 1, 3, 96),
    "many_requests": ([20000] + [(577 * i) % 900 for i in range(99)], [90 if i % 16 == 0 else 1 for i in range(100)], 32, 1, 4, 64),
}


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 0), (1500, 4), (4000, 4), (1500, 700), (2500, 130)])
@pytest.mark.parametrize("name", SPLIT)
def test_splits_of_a_window(name, window, sinks, act):
    """Splits that start among the first tokens, that hold the gap after them, and that end in the window."""
    s = R.case(*SPLIT[name], act, seed=window + sinks, device=DEV)
    got = _run(s, window=window, sinks=sinks)
    _check(s, window, sinks, got)
    assert torch.equal(_run(s, window=window, sinks=sinks), got)
    L.paged_check()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("requests", [64, 65, 128, 1025, 4096])
@pytest.mark.parametrize("dim,group,window,sinks", [(64, 1, 0, 0), (96, 2, 20, 3), (128, 2, 0, 0), (256, 1, 50, 0)])
def test_many_requests(requests, dim, group, window, sinks, act):
    """One wave's worth of requests, one more, and as many as a call takes; some without new tokens, some with a chunk."""
    few = 1 if requests < 1000 else 4
    cached = [(37 * i) % (400 // few) for i in range(requests)]
    new = [0 if i % 11 == 5 else 1 + (140 // few) * (i % 97 == 64) for i in range(requests)]
    s = R.case(cached, new, 16, 1, group, dim, act, device=DEV)
    _check(s, window, sinks, _run(s, window=window, sinks=sinks), _run(s, window=window, sinks=sinks, max_new=max(new)))
    L.paged_check()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("cached,new,page,group,dim,window", [
    (70, 5, 16, 2, 96, 0), (30, 200, 16, 2, 128, 0), (50, 150, 32, 1, 256, 20), (5000, 90, 64, 2, 64, 0), (5000, 90, 16, 2, 128, 1200),
    (20000, 4, 16, 4, 128, 0), (20000, 4, 64, 2, 256, 900), (3000, 130, 32, 2, 96, 60)])
def test_what_is_no_number_stays_with_who_sees_it(cached, new, page, group, dim, window, bad, act):
    """A key and a value in a later token's place, before a window and past the last token, in calls that split and in
    those that do not: rows that see neither are the definition's; a value that is seen shows where it is, and only there."""
    s = R.case([cached], [new], page, 1, group, dim, act, device=DEV)
    spots = [cached + new // 2] + ([cached - window, cached - window + 1] if window else [])
    sees = [any(cached + i >= p and (not window or cached + i - window < p) for p in spots) for i in range(new)]
    clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
    at = [(s["tables"][0][p // page], p % page) for p in spots]
    for pg, o in at:
        s["k"][pg, :, o] = bad
        s["v"][pg, :, ::3, o] = bad
    got = _run(s, window=window)
    want, *rest = _dense(clean, 0, window, 0)
    tol = R.bound(want, *rest, act, dim)
    off = (got.double().cpu() - want).abs()
    blind = torch.tensor([not x for x in sees])
    assert (off[blind] <= tol[blind]).all()
    # the value alone, where every value of the key is 1 but for one dimension
    for pg, o in at:
        s["k"][pg, :, o] = 0
        s["v"][pg, :, :, o] = 1
        s["v"][pg, :, 5, o] = bad
        clean["k"][pg, :, o] = 0
        clean["v"][pg, :, :, o] = 1
    got = _run(s, window=window)
    want, *rest = _dense(clean, 0, window, 0)
    tol = R.bound(want, *rest, act, dim)
    off = (got.double().cpu() - want).abs()
    rest = [d for d in range(dim) if d != 5]
    assert (off[..., rest] <= tol[..., rest]).all() and (off[blind] <= tol[blind]).all()
    assert not torch.isfinite(got[~blind.to(DEV)][..., 5]).any()
    L.paged_check()
