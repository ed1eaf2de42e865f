"""Calls whose launch would have 2^32 threads or more, whatever the tile, and calls whose outputs share memory with their inputs
are refused before anything is read or launched."""
import pytest

from .test_fp8_cpu import EINVAL, ESHAPE, PTR, _gate, _grouped, _matmul, _plan, _quantize, _weight, refused


@pytest.mark.parametrize("kw", [
    # 10 rows an expert: 4737 tiles of 64 rows at most, 3907 of 128 columns, 256 threads each
    dict(experts=4096, rows=40960, n=500000),
    dict(experts=4096, rows=40960, n=500000, out=1),
    dict(experts=4096, rows=40960, n=500000, dtype=30),
    # 5 rows: 5217 tiles of 32, 128 threads
    dict(experts=4096, rows=20480, n=1000000),
    # 4 rows: 5121 tiles of 16, 256 threads for 64 columns
    dict(experts=4096, rows=16384, n=300000),
    # 700 rows: 26497 tiles of 128, 256 threads for 128 columns
    dict(experts=4096, rows=2867200, n=100000),
    dict(experts=4096, rows=2867200, n=100000, out=1),
])
def test_grouped_launches_past_the_threads_of_a_grid(kw):
    sizes = dict(k=16, stride=16, xs_row=1, x_rows=kw["rows"], y_rows=kw["rows"])
    refused(_grouped, {**sizes, **kw}, ESHAPE, b"threads")


def test_a_launch_past_the_threads_of_a_grid():
    refused(_matmul, dict(m=1 << 23, n=1 << 16, k=16, stride=16, xs_row=1, y=PTR), ESHAPE, b"threads")


FAR = 1 << 30


@pytest.mark.parametrize("call,kw", [
    # f32 x [4, 256]: 4096 bytes; q 1024, scales 32
    (_quantize, dict(q=PTR + 4096 - 8, s=PTR + FAR)), (_quantize, dict(q=PTR - 1024 + 8, s=PTR + FAR)),
    (_quantize, dict(q=PTR + FAR, s=PTR + 4092)), (_quantize, dict(q=PTR + FAR, s=PTR + FAR + 1020)),
    (_quantize, dict(q=PTR + FAR, s=PTR + FAR - 28)), (_quantize, dict(q=PTR + 1 * FAR, s=PTR - 4 * 1000, ss=1000)),
    # f16: 2048 bytes
    (_gate, dict(u=PTR + FAR, q=PTR + 2040, s=PTR + 2 * FAR)), (_gate, dict(g=PTR + FAR, q=PTR, s=PTR + 2 * FAR)),
    (_gate, dict(u=PTR + FAR, q=PTR + 2 * FAR, s=PTR + FAR + 16)),
    # bf16 [2, 100, 256]: 102400 bytes, q 51200, scales 16
    (_weight, dict(q=PTR + 102400 - 8, s=PTR + FAR)), (_weight, dict(q=PTR + FAR, s=PTR + FAR + 51196)),
    # y [4, 100] f32: 1600 bytes; x 1024, scales of x 32, weight 25600, its scales 8
    (_matmul, dict(y=PTR + 1008, w=PTR + FAR, ws=PTR + 2 * FAR, xs=PTR + 3 * FAR)),
    (_matmul, dict(y=PTR + FAR + 25584, w=PTR + FAR, ws=PTR + 2 * FAR, xs=PTR + 3 * FAR)),
    (_matmul, dict(y=PTR + 2 * FAR - 1584, w=PTR + FAR, ws=PTR + 2 * FAR, xs=PTR + 3 * FAR)),
    (_matmul, dict(y=PTR + 3 * FAR + 16, w=PTR + FAR, ws=PTR + 2 * FAR, xs=PTR + 3 * FAR)),
    (_grouped, dict(y=PTR + FAR, w=PTR + 2 * FAR, ws=PTR + 3 * FAR, xs=PTR + 4 * FAR, starts=PTR + FAR + 1596)),
    (_grouped, dict(y=PTR + FAR, w=PTR + 2 * FAR, ws=PTR + 3 * FAR, xs=PTR + 4 * FAR, starts=PTR + 5 * FAR, gather=PTR + FAR)),
    (_grouped, dict(y=PTR + FAR, w=PTR + 2 * FAR, ws=PTR + 3 * FAR, xs=PTR + 4 * FAR, starts=PTR + 5 * FAR,
                    scatter=PTR + FAR - 12, y_rows=9)),
    (_grouped, dict(y=PTR + 2 * FAR + 4 * 25600 - 16, w=PTR + 2 * FAR, ws=PTR + 3 * FAR, xs=PTR + 4 * FAR, starts=PTR + 5 * FAR)),
    # 8 ids; 9 starts
    (_plan, dict(starts=PTR + 28, planes=PTR + FAR, of=PTR + 2 * FAR)), (_plan, dict(starts=PTR + FAR, planes=PTR + FAR + 32, of=PTR + 2 * FAR)),
    (_plan, dict(starts=PTR + FAR, planes=PTR + 2 * FAR, of=PTR + 2 * FAR))])
def test_outputs_that_share_memory(call, kw):
    refused(call, kw, EINVAL, b"overlap")
