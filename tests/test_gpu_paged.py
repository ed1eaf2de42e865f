"""The paged cache on the GPU against its definition in 64 bits (paged_ref)."""
import math

import pytest
import torch

import lloom_amd as L
from lloom_amd.lib import LloomHipError
from lloom_amd.quantized import reserve_workspace

from . import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, F32 = torch.float16, torch.float32


# ------------------------------------------------------------------- plan --

PLANS = {
    "one": ([0], [1], 0), "first_token_of_a_page": ([16], [1], 0), "prompt": ([0], [1000], 0),
    "mixed": ([0, 15, 16, 17, 400, 31], [33, 1, 1, 0, 1, 130], 0), "padded": ([3, 90], [1, 1], 6),
    "none_new": ([5, 7], [0, 0], 3), "many": (list(range(0, 300)), [(7 * i) % 5 for i in range(300)], 11),
    "a_thousand": ([(37 * i) % 900 for i in range(1025)], [1] * 1025, 0),
}


def _tables(cached, new, page, blocks):
    """Old pages from the top, free ones from the bottom, in no order."""
    at, tables = 100000, []
    for c in cached:
        row = []
        for _ in range(R.pages_for(c, page)):
            row.append(at)
            at -= 3
        tables.append(row + [0] * (blocks - len(row)))
    free = [(i * 7) % 99991 for i in range(1, 5 + sum(R.pages_for(c + n, page) - R.pages_for(c, page)
                                                      for c, n in zip(cached, new)))]
    return tables, free


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("name", PLANS)
@pytest.mark.parametrize("page", [16, 64])
def test_plan(name, page):
    cached, new, pad = PLANS[name]
    blocks = max(R.pages_for(c + n, page) for c, n in zip(cached, new)) + 2
    tables, free = _tables(cached, new, page, blocks)
    tokens = sum(new) + pad
    wide = torch.full((len(cached), blocks + 3), -7, dtype=torch.int32, device=DEV)
    wide[:, :blocks] = _ints(tables)
    got = L.paged_plan(_ints(cached), _ints(new), tokens, wide[:, :blocks], _ints(free), page)
    L.paged_check()
    start, lens, pos, slots, taken, after = R.plan(cached, new, tokens, tables, free, page)
    assert got.q_start.tolist() == start and got.seq_lens.tolist() == lens and got.taken.tolist() == [taken]
    assert got.positions.tolist() == pos and got.slots.tolist() == slots
    assert got.block_tables.tolist() == after and (wide[:, blocks:] == -7).all()


@pytest.mark.parametrize("cached,new,tokens,blocks,free", [
    ([0, 10], [40, 30], 70, 4, 3),     # too few free pages
    ([0, 10], [40, 60], 100, 4, 9),    # a table that is too short
    ([0, 10], [40, 6], 40, 4, 9),      # fewer rows than new tokens
    ([-1, 10], [40, 6], 46, 4, 9), ([1, 10], [40, -6], 46, 4, 9)])
def test_plan_reports_what_does_not_fit(cached, new, tokens, blocks, free):
    tables = [[50] + [0] * (blocks - 1), [60] + [0] * (blocks - 1)]
    got = L.paged_plan(_ints(cached), _ints(new), tokens, _ints(tables), _ints(list(range(1, free + 1))), 16)
    with pytest.raises(LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EPAGE"
    L.paged_check()
    c, n = [max(v, 0) for v in cached], [max(v, 0) for v in new]
    start, lens, pos, slots, taken, after = R.plan(c, n, tokens, tables, list(range(1, free + 1)), 16)
    assert got.q_start.tolist() == start and got.seq_lens.tolist() == lens and got.taken.tolist() == [taken]
    assert got.slots.tolist() == slots and got.block_tables.tolist() == after


# ----------------------------------------------------------------- append --

@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("page,heads,dim,slots", [
    (16, 2, 64, [5]), (16, 4, 128, [40, 3, -1, 17, 8, 9]), (32, 1, 256, list(range(37, 37 + 90))),
    (64, 3, 96, list(range(64, 192)) + [-1] * 5 + list(range(5, 30))),
    (16, 8, 128, [16 * ((7 * i) % 401) + i % 16 for i in range(401)]),
    (128, 16, 64, list(range(3, 1100)))])
def test_append(act, page, heads, dim, slots):
    g = torch.Generator(device=DEV).manual_seed(len(slots))
    pages, n = 402 if len(slots) == 401 else max(slots) // page + 2, len(slots)
    k0 = torch.randn(pages, heads, page, dim, generator=g, device=DEV).half()
    v0 = torch.randn(pages, heads, dim, page, generator=g, device=DEV).half()
    # k and v as slices of one projection's rows
    fused = (torch.randn(n, 3 * heads * dim, generator=g, device=DEV) * 100).to(act)
    k, v = fused[:, heads * dim:2 * heads * dim].view(n, heads, dim), fused[:, 2 * heads * dim:].view(n, heads, dim)
    kc, vc = k0.clone(), v0.clone()
    L.paged_append(kc, vc, k, v, torch.tensor(slots, device=DEV))
    L.paged_check()
    for i, s in enumerate(slots):
        if s >= 0:
            k0[s // page, :, s % page] = k[i].half()
            v0[s // page, :, :, s % page] = v[i].half()
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_append_values_and_layouts():
    """Infinities, NaN, values past f16's largest and subnormal ones are rounded as a cast; heads that are not dense and
    rows that are not 16-byte aligned are read too."""
    n, heads, dim = 9, 2, 64
    x = torch.randn(n, heads, dim, device=DEV)
    x[0, 0, :6] = torch.tensor([math.inf, -math.inf, 65520.0, -1e9, 3e-8, 2.0 ** -25], device=DEV)
    x[1, 1, 3] = math.nan
    want = x.half()
    slots = torch.arange(4, 4 + n, device=DEV)
    for t in (x, x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x[..., :1], x], -1)[..., 1:],
              torch.nn.functional.pad(x.reshape(n, -1), (1, 2))[:, 1:-2].view(n, heads, dim)):
        kc, vc = (torch.zeros(2, heads, 16, dim, dtype=F16, device=DEV), torch.zeros(2, heads, dim, 16, dtype=F16, device=DEV))
        L.paged_append(kc, vc, t, t, slots)
        got = torch.cat([kc[0], kc[1]], 1)[:, 4:4 + n].transpose(0, 1)
        assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
        got = torch.cat([vc[0], vc[1]], 2)[:, :, 4:4 + n].permute(2, 0, 1)
        assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
    L.paged_append(kc, vc, x[:0], x[:0], slots[:0])
    L.paged_check()


def test_append_leaves_out_a_slot_past_the_cache():
    kc, vc = torch.zeros(2, 1, 16, 64, dtype=F16, device=DEV), torch.zeros(2, 1, 64, 16, dtype=F16, device=DEV)
    x = torch.ones(3, 1, 64, device=DEV)
    L.paged_append(kc, vc, x, x, torch.tensor([31, 32, 1 << 40], device=DEV))
    with pytest.raises(LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EPAGE"
    assert kc.sum() == 64 and vc.sum() == 64 and (kc[1, 0, 15] == 1).all() and (vc[1, 0, :, 15] == 1).all()


# -------------------------------------------------------------- attention --

def _check(s, got, window=0, sinks=0, scale=None):
    want = R.attention(s["q"], s["k"], s["v"], s["tables"], s["q_start"], s["seq_lens"],
                       s["scale"] if scale is None else scale, window, sinks)
    tol = R.bound(*want, s["q"].dtype, s["q"].shape[-1])
    assert got.dtype == s["q"].dtype and got.shape == s["q"].shape
    off = (got.double().cpu() - want[0]).abs()
    assert torch.isfinite(got).all() and (off <= tol).all(), (off / tol).max()


def _run(s, **kw):
    return L.paged_attention(s["q"], s["k"], s["v"], s["t_tables"], s["t_start"], s["t_lens"], **kw)


#                   cached, new, page, kv_heads, group, dim
SHAPES = {
    "first_token": ([0], [1], 16, 1, 1, 64), "second_token": ([1], [1], 16, 2, 4, 128),
    "page_ends": ([14, 15, 16, 31, 32], [1] * 5, 16, 2, 2, 64), "long": ([5000], [1], 64, 2, 4, 128),
    "lengths": ([0, 1, 700, 127, 128, 129], [1] * 6, 32, 1, 8, 96), "wide_heads": ([300, 33], [1, 1], 128, 2, 3, 256),
    "sixteen_heads_a_key": ([77], [1], 16, 1, 16, 128), "forty_heads_a_key": ([77, 3], [1, 1], 16, 1, 40, 64),
    "few_new": ([40, 100], [3, 5], 16, 2, 3, 64), "prompt": ([0], [130], 16, 1, 2, 64),
    "ragged": ([0, 50, 0, 200], [67, 1, 0, 33], 16, 2, 1, 128), "odd_group": ([60], [41], 32, 1, 5, 96),
    "chunk_256": ([90, 10], [37, 64], 16, 1, 2, 256), "many": ([3 * i for i in range(70)], [1] * 70, 16, 1, 2, 64),
    "many_chunks": ([5 * i for i in range(80)], [1 + 40 * (i % 3 == 1) for i in range(80)], 16, 2, 2, 64),
    "chunk_long": ([1100], [140], 64, 1, 2, 128), "mixed": ([500, 0, 90, 7], [1, 200, 1, 1], 16, 1, 4, 128),
}


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("name", SHAPES)
def test_attention(name, act):
    s = R.case(*SHAPES[name], act, device=DEV)
    _check(s, _run(s))
    L.paged_check()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (33, 4), (100, 1), (64, 40), (5000, 4), (7, 300)])
@pytest.mark.parametrize("name", ["lengths", "few_new", "ragged", "chunk_long", "mixed"])
def test_attention_window(name, window, sinks, act):
    s = R.case(*SHAPES[name], act, seed=window, device=DEV)
    _check(s, _run(s, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("name", ["lengths", "mixed", "ragged", "few_new"])
def test_max_new_only_tells(name, act):
    """The results stand with the longest chunk told, not told, and told wrong."""
    s = R.case(*SHAPES[name], act, device=DEV)
    for n in (max(SHAPES[name][1]), 1, 100000):
        _check(s, _run(s, max_new=n))


@pytest.mark.parametrize("act", [F32, F16])
def test_attention_arguments(act):
    """Another scale, rows of q that are slices of a fused projection, heads that are not dense, an output given."""
    s = R.case([50, 9], [1, 20], 16, 2, 2, 64, act, device=DEV)
    n, heads, dim = s["q"].shape
    _check(s, _run(s, scale=0.3), scale=0.3)
    _check(s, _run(s, scale=-0.2), scale=-0.2)
    _check(s, _run(s, scale=0.0), scale=0.0)
    many = R.case([500], [70], 16, 1, 2, 64, act, device=DEV)
    for scale in (0.0, -0.3):
        _check(many, _run(many, scale=scale), scale=scale)
    q, same = s["q"], _run(s)
    fused = torch.zeros(n, 2 * heads * dim, dtype=act, device=DEV)
    fused[:, :heads * dim] = q.reshape(n, -1)
    apart = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty_like(same)
    for t in (fused[:, :heads * dim].view(n, heads, dim), apart):
        s["q"] = t
        assert torch.equal(_run(s, out=out), same)
    with pytest.raises(LloomHipError):
        _run(s, out=out[:, :1])


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("top", [1e-6, 1.0, 200.0, 30000.0])
def test_attention_magnitudes(act, top):
    """Scores from nearly equal ones to a single key that takes all the weight, and values up to f16's largest."""
    s = R.case([300], [9], 16, 1, 2, 64, F32, device=DEV)
    s["q"] = (s["q"] * top).clamp(-60000.0, 60000.0).to(act)  # finite in either type
    s["v"].mul_(10000.0)
    scale = 0.125 * min(1.0, 1.0 / top) * 8
    _check(s, _run(s, scale=scale), scale=scale)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_that_see_nothing_are_zero(act, dim):
    s = R.case([40, 0, 3, 0], [1, 0, 2, 70], 16, 2, 2, dim, act, pad=5, device=DEV)
    got = _run(s)
    _check(s, got)
    assert (got[-5:] == 0).all()
    # more new tokens than the lengths say: the first rows are at negative positions
    s["seq_lens"] = [20, 0, 1, 30]
    s["t_lens"] = _ints(s["seq_lens"])
    got = _run(s)
    _check(s, got)
    assert (got[1] == 0).all() and (got[3:43] == 0).all() and (got[43] != 0).any()
    s["t_lens"] = _ints([0, -5, 0, -2147483648])
    assert (_run(s) == 0).all()
    L.paged_check()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("name", ["lengths", "chunk_long", "mixed"])
def test_bad_pages_are_passed_over_and_reported(name, act):
    s = R.case(*SHAPES[name], act, device=DEV)
    pages = s["k"].shape[0]
    for b, bad in ((0, -1), (len(s["tables"]) - 1, pages), (2 % len(s["tables"]), 1 << 30)):
        row = s["tables"][b]
        used = R.pages_for(s["seq_lens"][b], s["k"].shape[2])
        row[used // 2] = bad
    s["t_tables"] = _ints(s["tables"])
    got = _run(s)
    _check(s, got)
    with pytest.raises(LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EPAGE"


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("cached,new,dim", [(900, 1, 64), (900, 70, 128), (900, 40, 256), (300, 300, 96)])
def test_pages_that_no_token_sees_may_be_none(cached, new, dim, act):
    """A server frees the pages between the first tokens and the window: nothing is read or reported there."""
    window, sinks, page = 100, 5, 16
    s = R.case([cached, 20], [new, 3], page, 2, 2, dim, act, device=DEV)
    want = _run(s, window=window, sinks=sinks)
    for i in range(len(s["tables"][0])):
        if i * page >= sinks and (i + 1) * page <= cached - window + 1:
            s["tables"][0][i] = -1
    assert -1 in s["tables"][0]
    s["t_tables"] = _ints(s["tables"])
    got = _run(s, window=window, sinks=sinks)
    L.paged_check()
    assert torch.equal(got, want)
    _check(s, got, window, sinks)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("cached,new,page,group", [(0, 1, 16, 64), (63, 65, 16, 1), (1000, 129, 32, 1), (127, 16, 4096, 8),
                                                   (2500, 33, 128, 4), (5, 260, 16, 3)])
def test_attention_of_one_chunk(cached, new, page, group, dim, act):
    """One request, in whichever way its rows and keys are cut: tiles and steps that are just full, and just over."""
    s = R.case([cached], [new], page, 2, group, dim, act, seed=new, device=DEV)
    _check(s, _run(s, max_new=new))
    _check(s, _run(s, window=77, sinks=3), 77, 3)
    L.paged_check()


#                   cached, new, page, kv_heads, group, dim
LONG = {
    "tiles_and_splits": ([6000], [512], 64, 4, 4, 64), "splits_of_a_few_rows": ([30000], [9], 16, 1, 4, 128),
    "one_long_among_short": ([20000, 40, 0, 700], [300, 64, 129, 1], 32, 2, 4, 64),
    "more_tiles_than_the_card_holds": ([0, 900], [3000, 1100], 128, 8, 4, 64),
    "splits_of_rows_beside_splits_of_tiles": ([30000, 20000, 25000, 9000], [1, 300, 2, 1], 32, 2, 4, 64),
    "many_requests": ([(911 * i) % 1500 for i in range(321)], [0 if i % 7 == 3 else 1 for i in range(321)], 32, 1, 4, 64),
    "many_requests_and_chunks": ([20000] + [(577 * i) % 900 for i in range(129)], [90 if i % 16 == 0 else 1 for i in range(130)], 32, 1, 4, 64),
    "long_and_short_tokens": ([60000, 3, 900, 33], [1, 1, 1, 1], 16, 2, 8, 128),
}


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("name", LONG)
def test_long_requests_in_splits(name, act):
    """Every way a call's tiles and splits are dealt out, each request against the definition, and the same twice."""
    s = R.case(*LONG[name], act, device=DEV)
    got = _run(s)
    L.paged_check()
    assert all(torch.equal(_run(s), got) for _ in range(20))
    for b in range(len(s["seq_lens"])):
        out, *rest = R.dense(s, b)
        tol = R.bound(out, *rest, act, s["q"].shape[-1])
        off = (got[s["q_start"][b]:s["q_start"][b + 1]].double().cpu() - out).abs()
        assert (off <= tol).all(), (b, (off / tol).max())


@pytest.mark.parametrize("act", [F32, F16])
def test_lengths_past_the_tables_are_reported(act):
    s = R.case([90], [20], 16, 1, 2, 64, act, device=DEV)
    s["tables"] = [s["tables"][0][:3]]
    s["t_tables"] = s["t_tables"][:, :3]
    for window in (0, 10):
        _check(s, _run(s, window=window), window)
        with pytest.raises(LloomHipError):
            L.paged_check()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("cached,new,group,window", [(0, 9, 1, 0), (70, 5, 2, 0), (30, 200, 2, 0), (50, 150, 1, 20)])
def test_what_a_token_does_not_see_may_be_anything(cached, new, group, window, bad, act):
    """A key and a value that are no numbers, in a later token's place and before a window, leave the others alone."""
    s = R.case([cached], [new], 16, 1, group, 64, act, device=DEV)
    clean = _run(s, window=window)
    p = cached + new // 2  # the position that is spoilt
    pg = s["tables"][0][p // 16]
    s["k"][pg, :, p % 16] = bad
    s["v"][pg, :, ::3, p % 16] = bad
    got = _run(s, window=window)
    sees = [cached + i >= p and (not window or cached + i - window < p) for i in range(new)]
    for i, see in enumerate(sees):
        if not see:
            assert torch.equal(got[i], clean[i]), i
    # one that sees the value alone takes it up
    s["k"][pg, :, p % 16] = 0
    s["v"][pg, :, :, p % 16] = 1
    s["v"][pg, :, 5, p % 16] = bad
    got = _run(s, window=window)
    for i, see in enumerate(sees):
        assert torch.isfinite(got[i, :, 5]).all() != see, i
        assert torch.isfinite(got[i, :, 6]).all()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("new", [1, 90])
def test_offsets_past_32_bits(act, new):
    """Pages at both ends of a cache of over 2^31 elements."""
    small = R.case([100], [new], 64, 8, 2, 128, act, device=DEV)
    per = 8 * 64 * 128
    pages = (1 << 31) // per + 500
    s = dict(small)
    s["k"] = torch.empty(pages, 8, 64, 128, dtype=F16, device=DEV)
    s["v"] = torch.empty(pages, 8, 128, 64, dtype=F16, device=DEV)
    homes = [pages - 1 - 7 * i for i in range(small["k"].shape[0])]
    for i, h in enumerate(homes):
        s["k"][h], s["v"][h] = small["k"][i], small["v"][i]
    s["t_tables"] = _ints([[homes[p] if p < len(homes) else p for p in row] for row in small["tables"]])
    assert torch.equal(_run(s), _run(small))
    rows = torch.randn(2, 8, 128, device=DEV).to(act)
    L.paged_append(s["k"], s["v"], rows, rows, torch.tensor([pages * 64 - 1, 5], device=DEV))
    assert torch.equal(s["k"][-1, :, -1], rows[0].half()) and torch.equal(s["v"][-1, :, :, -1], rows[0].half())
    assert torch.equal(s["v"][0, :, :, 5], rows[1].half())


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("name", ["long", "mixed", "chunk_long"])
def test_runs_are_alike_on_any_stream(name, act):
    s = R.case(*SHAPES[name], act, device=DEV)
    want = _run(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [_run(s) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("act", [F32, F16])
def test_a_captured_step_follows_the_lengths(act):
    """Plan, append and attention captured once and replayed as the requests grow, against eager calls."""
    heads, group, dim, page, n = 2, 2, 64, 16, 3
    cached = torch.tensor([0, 15, 100], dtype=torch.int32, device=DEV)
    new = torch.ones(n, dtype=torch.int32, device=DEV)
    cache = L.PagedCache(64, page, heads, dim)
    cache.k.normal_(), cache.v.normal_()
    tables = torch.zeros(n, 12, dtype=torch.int32, device=DEV)
    tables[:, :7] = torch.arange(21, dtype=torch.int32, device=DEV).view(n, 7)
    free = torch.arange(30, 60, dtype=torch.int32, device=DEV)
    q, k, v = (torch.zeros(n, h, dim, dtype=act, device=DEV) for h in (heads * group, heads, heads))
    reserve_workspace(L.paged_attention_workspace_bytes(n, n, heads, group, dim, 1))

    def step():
        plan = L.paged_plan(cached, new, n, tables, free, page)
        cache.append(k, v, plan.slots)
        return cache.attention(q, plan, window=50, sinks=2, max_new=1), plan.slots

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, slots = step()
    for i in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got, at, caches = out.clone(), slots.clone(), (cache.k.clone(), cache.v.clone())
        want, want_at = step()
        assert torch.equal(got, want) and torch.equal(at, want_at)
        assert torch.equal(caches[0], cache.k) and torch.equal(caches[1], cache.v)
        cached += 1
    L.paged_check()


def test_a_capture_without_workspace_is_refused():
    import lloom_amd.quantized as Q
    from lloom_amd.lib import check, lib
    import ctypes

    s = R.case([300], [1], 16, 2, 2, 64, F16, device=DEV)
    p = ctypes.c_void_p()
    check(lib().lloom_hip_ctx_create(0, ctypes.byref(p)))
    old = Q._ctxs.get(0)
    Q._ctxs[0] = p.value
    try:
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(LloomHipError) as e:
            with torch.cuda.graph(graph):
                _run(s)
        assert e.value.name == "ENOMEM"
    finally:
        if old is None:
            del Q._ctxs[0]
        else:
            Q._ctxs[0] = old
        torch.cuda.synchronize()
        check(lib().lloom_hip_ctx_destroy(p))
    _check(s, _run(s))


def test_prompt_in_chunks_and_then_tokens():
    """A prompt read in three chunks and then decoded, through the cache's own calls, is causal attention over all."""
    heads, group, dim, page = 2, 2, 64, 16
    n = 60
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV) for h in (heads * group, heads, heads))
    cache = L.PagedCache(9, page, heads, dim)
    tables = torch.zeros(1, 5, dtype=torch.int32, device=DEV)
    free = torch.tensor([4, 0, 8, 2, 7], dtype=torch.int32, device=DEV)
    got, done = [], 0
    for m in (25, 1, 30, 1, 1, 1, 1):
        plan = L.paged_plan(_ints([done]), _ints([m]), m, tables, free, page)
        cache.append(k[done:done + m], v[done:done + m], plan.slots)
        got.append(cache.attention(q[done:done + m], plan, max_new=m))
        free = free[int(plan.taken):]
        done += m
    L.paged_check()
    s = {"q": q, "k": cache.k, "v": cache.v, "tables": tables.tolist(), "q_start": [0, n], "seq_lens": [n],
         "scale": 1 / math.sqrt(dim)}
    _check(s, torch.cat(got))


def test_a_layer_of_packed_projections_over_the_cache():
    """The example's server: chunks of prompts beside decoding requests, against each whole request at once.  Scores of
    unit normal q and k are off by at most sum |q||k| / sqrt(128) (about 7.2) times 136 half f32 steps and 2^-21 (see
    paged_ref.bound), 6e-5, on either side: outputs by d = 1.2e-4 of their size.  The output projection takes them in 8-bit
    blocks, of steps s = 1/127 of a block's largest, about 3 / 127 of its size: a value changes its step with a
    probability of d / s and then by s, so that the norm is off by sqrt(d s) = 1.7e-3 at most."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_layer.py")
    spec = importlib.util.spec_from_file_location("paged_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    worst, us = example.run(prompts=(300, 37, 130, 1), steps=12, chunk=128)
    assert us is not None and worst < 1.7e-3
