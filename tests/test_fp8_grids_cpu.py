"""Calls whose launch would have 2^32 threads or more are refused before anything is read or launched, whatever the tile."""
import pytest

from .test_fp8_cpu import ESHAPE, PTR, _grouped, _matmul, refused


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
