"""The paged cache's refusals, which need no GPU: every call below is refused before anything is read."""
import ctypes

import pytest
import torch

import lloom_amd as L
from lloom_amd.lib import LloomHipError, lib

from . import paged_ref as R

PTR = 1 << 20  # a 16-byte aligned address that nothing reads


def _plan(**kw):
    a = dict(ctx=PTR, cached=PTR, new=PTR, requests=2, tokens=8, tables=PTR, stride=4, blocks=4, free=PTR, free_count=3,
             page=16, start=PTR, lens=PTR, pos=PTR, slots=PTR, taken=PTR, stream=None)
    a.update(kw)
    return lib().lloom_hip_paged_plan(*a.values())


def _append(**kw):
    a = dict(ctx=PTR, act=0, k=PTR, ks=256, v=PTR, vs=256, slots=PTR, tokens=4, kc=PTR, vc=PTR, pages=8, heads=2, dim=128,
             page=16, stream=None)
    a.update(kw)
    return lib().lloom_hip_paged_append(*a.values())


def _attend(**kw):
    a = dict(ctx=PTR, act=0, q=PTR, qs=1024, tokens=4, kc=PTR, vc=PTR, pages=8, heads=2, group=4, dim=128, page=16,
             tables=PTR, stride=4, blocks=4, start=PTR, lens=PTR, requests=2, scale=0.1, window=0, sinks=0, max_new=0,
             out=PTR, stream=None)
    a.update(kw)
    return lib().lloom_hip_paged_attention(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), 1), (dict(cached=None), 1), (dict(pos=None), 1), (dict(free=None), 1), (dict(requests=0), 1),
    (dict(tokens=-1), 1), (dict(blocks=0), 1), (dict(requests=4097), 3), (dict(stride=3), 3), (dict(page=8), 3),
    (dict(page=48), 3), (dict(page=8192), 3), (dict(tokens=1 << 31), 3)])
def test_plan_refusals(kw, code):
    assert _plan(**kw) == code
    assert b"paged_plan" in lib().lloom_hip_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), 1), (dict(k=None), 1), (dict(slots=None), 1), (dict(act=12), 2), (dict(dim=80), 3), (dict(page=20), 3),
    (dict(pages=0), 1), (dict(heads=0), 1), (dict(ks=255), 3), (dict(vs=128), 3), (dict(k=PTR + 4), 1), (dict(vs=258), 1),
    (dict(act=1, ks=260), 1), (dict(vc=PTR + 2), 1), (dict(tokens=-1), 1)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code
    assert b"paged_append" in lib().lloom_hip_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), 1), (dict(q=None), 1), (dict(lens=None), 1), (dict(act=8), 2), (dict(dim=32), 3), (dict(page=17), 3),
    (dict(pages=0), 1), (dict(group=0), 1), (dict(requests=0), 1), (dict(requests=5000), 3), (dict(stride=3), 3),
    (dict(blocks=0), 3), (dict(qs=1023), 3), (dict(q=PTR + 8), 1), (dict(out=PTR + 4), 1), (dict(window=-1), 1),
    (dict(sinks=-2), 1), (dict(scale=float("inf")), 1), (dict(scale=float("nan")), 1), (dict(max_new=-1), 1),
    (dict(tokens=1 << 30), 3), (dict(qs=1026), 1)])
def test_attention_refusals(kw, code):
    assert _attend(**kw) == code
    assert b"paged_attention" in lib().lloom_hip_last_error()


def test_workspace_bytes():
    few = L.paged_attention_workspace_bytes(32, 32, 4, 4, 128)
    assert 0 < few < 64 << 20
    assert L.paged_attention_workspace_bytes(32, 32, 4, 4, 128, max_new=1) <= few
    out = ctypes.c_size_t()
    f = lib().lloom_hip_paged_attention_workspace_bytes
    assert f(32, 32, 4, 4, 80, 0, ctypes.byref(out)) == 3 and f(32, 0, 4, 4, 128, 0, ctypes.byref(out)) == 1
    assert f(32, 32, 4, 4, 128, 0, None) == 1


@pytest.mark.parametrize("kw", [dict(head_dim=80), dict(page_size=24), dict(pages=0), dict(kv_heads=0)])
def test_cache_refusals(kw):
    a = dict(pages=2, page_size=16, kv_heads=2, head_dim=64, device="cpu")
    a.update(kw)
    with pytest.raises(LloomHipError):
        L.PagedCache(**a)


def test_tensor_refusals():
    """Shapes, types and layouts that the Python calls refuse by name before the library is asked."""
    s = R.case([5, 0], [1, 3], 16, 2, 2, 64, torch.float32)
    ok = (s["q"], s["k"], s["v"], s["t_tables"], s["t_start"], s["t_lens"])

    def refused(i, t, code):
        a = list(ok)
        a[i] = t
        with pytest.raises(LloomHipError) as e:
            L.paged_attention(*a)
        assert e.value.code == code, e.value

    refused(0, s["q"][:, :3], 3)                      # heads not a multiple
    refused(0, s["q"][..., :32], 3)                   # another head_dim
    refused(0, s["q"].bfloat16(), 2)
    refused(1, s["k"].float(), 3)
    refused(1, s["k"].transpose(2, 3), 3)
    refused(2, s["k"], 3)                             # v in k's layout
    refused(3, s["t_tables"].long(), 1)
    refused(3, s["t_tables"][:1], 3)
    refused(4, s["t_start"][:-1], 3)
    refused(5, s["t_lens"].float(), 1)
    with pytest.raises(LloomHipError):                # no CPU fallback
        L.paged_attention(*ok)
    with pytest.raises(LloomHipError) as e:
        L.paged_append(s["k"], s["v"], s["q"][:, :2], s["q"][:, :2].half(), torch.zeros(4, dtype=torch.int64))
    assert e.value.code == 2
    with pytest.raises(LloomHipError) as e:
        L.paged_append(s["k"], s["v"], s["q"][:, :2], s["q"][:, :2], torch.zeros(3, dtype=torch.int64))
    assert e.value.code == 3


def test_reference_plan_by_hand():
    start, lens, pos, slots, taken, tables = R.plan([16, 0, 5], [1, 17, 0], 20, [[9, 0], [0, 0], [4, 0]], [7, 2, 3], 16)
    assert start == [0, 1, 18, 18] and lens == [17, 17, 5] and taken == 3
    assert tables == [[9, 7], [2, 3], [4, 0]]
    assert pos[0] == 16 and slots[0] == 7 * 16 and slots[1] == 32 and slots[17] == 48 and slots[18:] == [-1, -1]
