"""What the products' sums hold: by default every type of y is the same f32 sums of exact products, rounded once, however many
rows share a call; with set_fp8_mma(MMA_FP8) halves of many rows may lose what fp8_ref.product's groups of eight allow."""
import numpy as np
import pytest
import torch

from . import fp8_ref as R
from .test_gpu_fp8 import ACTS, BF16, F16, F32, L, f64, normal, ragged, weights  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def fp8_mma(L):
    L.set_fp8_mma(L.MMA_FP8)
    yield
    L.set_fp8_mma(L.MMA_F16)


def check_rows(y, q, sx, w, ws, rows, groups8=False):
    """Rows `rows` of y against those of e4m3 q with scales sx times w, by the bound that fp8_ref.product derives."""
    want, off = R.product(R.values(q[rows]), f64(sx[rows]), R.values(w), f64(ws), y.dtype, groups8)
    err = np.abs(f64(y[rows]) - want)
    assert np.all(err <= off), (np.max(err / off), np.unravel_index(np.argmax(err / off), off.shape))


def sample(m, seed, count=24):
    """Rows around every place where a tile of rows may end, the first and the last among them, as far as they are few."""
    g = torch.Generator().manual_seed(seed)
    edges = [0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 255, 256, m - 2, m - 1]
    return torch.unique(torch.tensor([r for r in edges if 0 <= r < m] + torch.randint(m, (count,), generator=g).tolist()))


def cancelling(k):
    """A row of x and one of the weight whose large products meet their negatives among eight neighbours: what is left is 6 *
    24 of every eight, whole numbers that f32 sums hold in any order (none passes 2^24)."""
    x, w = torch.ones(k), torch.full((k,), 24.0)
    x[0::8] = x[1::8] = 448.0
    w[0::8], w[1::8] = 448.0, -448.0
    return x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn), 144.0 * (k // 8)


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("n", [264, 4100])
@pytest.mark.parametrize("m", [1, 16, 17, 64, 130, 300, 700, 2100])
def test_neighbours_that_cancel(L, m, n, out):
    for k, scale in ((256, 1.0), (2048, 0.125)):  # 4608, which all three types have, from both
        x, w, left = cancelling(k)
        ws = torch.full((-(-n // 128), k // 128), scale, device="cuda")
        y = L.fp8_matmul(x.expand(m, k).cuda(), w.expand(n, k).contiguous().cuda(), ws,
                         x_scales=torch.ones(m, k // 128, device="cuda"), out_dtype=out)
        assert torch.all(y == left * scale)


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("each", [1, 3, 12, 100, 600])
def test_neighbours_that_cancel_by_expert(L, each, out):
    x, w, left = cancelling(256)
    E, n = 4, 264
    starts = (torch.arange(E + 1) * each).int().cuda()
    y = L.fp8_grouped_matmul(x.expand(E * each, 256).cuda(), w.expand(E, n, 256).contiguous().cuda(),
                             torch.ones(E, 3, 2, device="cuda"), starts, x_scales=torch.ones(E * each, 2, device="cuda"),
                             out_dtype=out)
    assert torch.all(y == left)


# (m, n, k) of every kernel and tile by number of steps: few rows; 32 x 128 and 64 x 128 with k in one part and in two; 128 x 128
# in two parts and in one, with one step, some, and past the 64 blocks whose scales a wave holds; ends inside tiles
SHAPES = [(3, 264, 656), (16, 4104, 2064), (64, 4096, 656), (17, 257, 1040), (128, 2050, 8336),  # few rows
          (300, 3001, 400), (700, 1000, 400), (600, 1000, 16), (20, 35000, 1040),  # 32 x 128
          (300, 3001, 1040), (200, 3100, 8336),      # 32 x 128, two parts
          (1400, 1500, 656), (700, 5000, 400), (1030, 1000, 272), (50, 40000, 272),  # 64 x 128
          (540, 2900, 1168), (400, 4200, 8208),      # 64 x 128, two parts
          (700, 4100, 4112), (1000, 4001, 2192),     # 128 x 128, two parts
          (3400, 3101, 656), (2304, 8200, 1168), (2500, 2100, 8336), (20000, 300, 1264), (5000, 1300, 16), (3000, 1800, 272), (100, 40000, 272)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_one_sum_for_all_types(L, m, n, k):
    w, ws = weights(n + k, n, k)
    q, sx = L.fp8_quantize(normal(m, m, k).cuda())
    y = L.fp8_matmul(q, w.cuda(), ws.cuda(), x_scales=sx)
    assert y.dtype is F32
    check_rows(y, q.cpu(), sx, w, ws, sample(m, k))
    for out in (F16, BF16):
        got = L.fp8_matmul(q, w.cuda(), ws.cuda(), x_scales=sx, out_dtype=out)
        assert torch.equal(got, y.to(out))


def grouped_sums(L, counts, extra, n, k, out, groups8):
    """Rows gathered and scattered, with rows of no expert, and the same from f32 x; returns what the plain call gave."""
    E = len(counts)
    starts, rows, order = ragged(counts, extra, E)
    w, ws = weights(E + n, E, n, k)
    tokens = rows // 2 + 1
    x = normal(rows, tokens, k)
    gather, scatter = (order % tokens).int(), torch.randperm(rows, generator=torch.Generator().manual_seed(1)).int()
    q, sx = L.fp8_quantize(x.cuda())
    args = (w.cuda(), ws.cuda(), starts.cuda())
    y = L.fp8_grouped_matmul(q, *args, x_scales=sx, gather=gather.cuda(), scatter=scatter.cuda(), out_dtype=out)
    plain = L.fp8_grouped_matmul(q[gather.long().cuda()], *args, x_scales=sx[gather.long().cuda()], out_dtype=out)
    assert torch.equal(y[scatter.long().cuda()], plain)
    assert torch.equal(L.fp8_grouped_matmul(x.cuda(), *args, gather=gather.cuda(), out_dtype=out), plain)
    assert not plain[int(starts[-1]):].any()
    L.paged_check()
    qg, sg, got = q.cpu()[gather.long()], sx.cpu()[gather.long()], plain.cpu()
    for e, c in enumerate(counts):
        if c:
            i = int(starts[e])
            check_rows(got[i:i + c], qg[i:i + c], sg[i:i + c], w[e], ws[e], sample(c, e, 6), groups8)
    return plain


COUNTS = [[1, 0, 2, 1, 0, 4, 3], [3, 9, 0, 14, 2, 7, 5], [16, 40, 0, 33, 64, 65, 15, 1], [250, 0, 129, 128, 127, 1],
          [513, 0, 700, 1030, 1, 900], [2049, 0, 3, 256], [600, 600, 600, 600, 512, 513, 511, 1025, 0]]
LONG = [[6000, 0, 9000, 13001, 512, 12600], [3000, 0, 5001, 4100, 700, 1500]]
# (groups, some empty and some that end inside a tile; n, k) of every kernel and tile, with one step, some, and over 64
GROUPED = [(COUNTS[0], 700, 656), (COUNTS[1], 264, 1168), (COUNTS[2], 257, 8336), (COUNTS[3], 129, 656), ([3] * 300, 600, 272),  # few
           (COUNTS[1], 4100, 400), (COUNTS[3], 700, 656), (COUNTS[5], 264, 16), ([7, 0, 9] * 90, 1500, 2064),  # 32 x 128
           (COUNTS[1], 4100, 1168), (COUNTS[3], 264, 1168), (COUNTS[5], 257, 8336),  # the same, two parts
           (COUNTS[4], 264, 656), (COUNTS[6], 700, 400), (COUNTS[3], 2200, 16), (COUNTS[4], 1280, 8336),  # 64 x 128
           (COUNTS[6], 257, 1168), (COUNTS[4], 384, 8336),  # the same, two parts
           (COUNTS[4], 2200, 400), (COUNTS[6], 2200, 1168), (LONG[0], 200, 272), (LONG[1], 700, 656),  # 128 x 128
           (COUNTS[4], 700, 2192), (COUNTS[5], 900, 8336)]  # the same, two parts


@pytest.mark.parametrize("counts,n,k", GROUPED)
def test_one_sum_for_all_types_by_expert(L, counts, n, k):
    y = grouped_sums(L, counts, 9, n, k, F32, False)
    for out in (F16, BF16):
        assert torch.equal(grouped_sums(L, counts, 9, n, k, out, False), y.to(out))


@pytest.mark.parametrize("m", [1, 16, 17, 64, 129, 600, 2100])
def test_a_row_is_the_same_to_f32_rounding_whatever_rows_share_its_call(L, m):
    """Two orders of summing a row are each within the bound of f32 sums, so no further apart than twice that."""
    n, k = 1030, 2064
    w, ws = weights(1, n, k)
    q, sx = L.fp8_quantize(normal(2, 2100, k).cuda())
    one = L.fp8_matmul(q[:1], w.cuda(), ws.cuda(), x_scales=sx[:1])
    got = L.fp8_matmul(q[:m], w.cuda(), ws.cuda(), x_scales=sx[:m].t().contiguous().t())[:1]
    _, off = R.product(R.values(q[:1]), f64(sx[:1]), R.values(w), f64(ws), F32, False)
    assert np.all(np.abs(f64(one) - f64(got)) <= 2 * off)


# ------------------------------------------------------------------ MMA_FP8 --

# the same with MMA_FP8: 32 x 128, the two parts, 64 x 128, 128 x 128, and 256 x 256 with 1, 2, 3, 6 and over 64 steps, where
# slots are filled again and scales read again; remainders in m, n and k
CUT_SHAPES = [(300, 3001, 400), (300, 3001, 1040), (1400, 1500, 656), (540, 2900, 1168), (700, 4100, 4112), (2304, 8200, 656),
              (3400, 3101, 16), (3400, 3101, 256), (3400, 3101, 272), (3400, 3101, 656), (3400, 3101, 8336), (4160, 8192, 400)]


@pytest.mark.parametrize("out", [F16, BF16])
@pytest.mark.parametrize("m,n,k", CUT_SHAPES)
def test_cut_sums(L, fp8_mma, m, n, k, out):
    """Within the bound value by value; and in the 2-norm the sums e are held to 3e-5 of the result, twice what normal values
    have.  y is rounded after, so that a value differs from the uncut one's by a step with a likelihood of |e| / step: sum of
    |e| step <= |e| |step|, and with steps of 2 * EPS of a value at most the difference is sqrt(3e-5 * 2 EPS) of the
    result in the 2-norm."""
    w, ws = weights(n + k, n, k)
    q, sx = L.fp8_quantize(normal(m, m, k).cuda())
    y = L.fp8_matmul(q, w.cuda(), ws.cuda(), x_scales=sx, out_dtype=out)
    check_rows(y, q.cpu(), sx, w, ws, sample(m, k), True)
    L.set_fp8_mma(L.MMA_F16)
    uncut = L.fp8_matmul(q, w.cuda(), ws.cuda(), x_scales=sx, out_dtype=out)
    far = (y.float() - uncut.float()).norm() / uncut.float().norm()
    assert 0 < far <= (3e-5 * 2 * R.EPS[out]) ** 0.5


# by expert, with MMA_FP8: a tile of each size, and (256, 256) by one, three and nine tiles of n, whose tiles of rows are no
# multiple of the four that are walked together nor of the eight XCDs, with 1, 2, 3, 6 and over 64 steps
CUT_GROUPED = [(COUNTS[3], 700, 656), (COUNTS[3], 264, 1168), (COUNTS[4], 264, 656), (COUNTS[6], 257, 1168), (COUNTS[4], 2200, 400),
               (COUNTS[5], 900, 8336), (LONG[0], 200, 272), (LONG[0], 256, 16), (LONG[1], 700, 656), (LONG[1], 641, 256),
               (COUNTS[6], 2200, 656), (COUNTS[6], 2200, 8336)]


@pytest.mark.parametrize("out", [F16, BF16])
@pytest.mark.parametrize("counts,n,k", CUT_GROUPED)
def test_cut_sums_by_expert(L, fp8_mma, counts, n, k, out):
    grouped_sums(L, counts, 9, n, k, out, True)


@pytest.mark.parametrize("counts,n", [(COUNTS[6], 2200), (LONG[0], 200), (LONG[1], 700)])
@pytest.mark.parametrize("starts", [[1, 2, 3], [0, 5, 3], [0, -1, 3], [0, 2, 1 << 30]])
def test_cut_sums_of_starts_out_of_order(L, fp8_mma, counts, n, starts):
    """On tiles of (256, 256)."""
    w, ws = weights(2, len(counts), n, 272)
    rows = sum(counts)
    bad = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32)
    bad[:3] = torch.tensor(starts, dtype=torch.int32)
    y = L.fp8_grouped_matmul(normal(3, rows, 272, dtype=F16).cuda(), w.cuda(), ws.cuda(), bad.cuda())
    with pytest.raises(L.LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EEXPERT" and y.shape == (rows, n) and not y.any()
    L.paged_check()


def test_into_f32_and_of_few_rows_nothing_is_cut(L, fp8_mma):
    x, w, left = cancelling(256)
    for m, out in ((3, F16), (64, BF16), (600, F32), (2100, F32)):
        y = L.fp8_matmul(x.expand(m, 256).cuda(), w.expand(264, 256).contiguous().cuda(), torch.ones(3, 2, device="cuda"),
                         x_scales=torch.ones(m, 2, device="cuda"), out_dtype=out)
        assert torch.all(y == left)


def test_modes_that_are_none_are_refused(L):
    for mode in (1, 2, 4, -1):
        with pytest.raises(L.LloomHipError) as e:
            L.set_fp8_mma(mode)
        assert e.value.name == "EINVAL"


# ------------------------------------------------------------------- sizes --

def test_many_experts_of_few_rows_by_a_long_n(L):
    """4096 experts of four rows each by 32768 columns: within a launch's threads with the tiles that serve them."""
    E, n, k = 4096, 32768, 16
    w = torch.randint(0, 0x60, (E, n, k), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ws = torch.rand(E, n // 128, 1, device="cuda")
    q, sx = L.fp8_quantize(normal(1, 4 * E, k).cuda())
    y = L.fp8_grouped_matmul(q, w, ws, (4 * torch.arange(E + 1)).int().cuda(), x_scales=sx, out_dtype=F16)
    for e in (0, 1, 2047, E - 1):
        check_rows(y[4 * e:4 * e + 4].cpu(), q[4 * e:4 * e + 4].cpu(), sx[4 * e:4 * e + 4], w[e].cpu(), ws[e], torch.arange(4))
