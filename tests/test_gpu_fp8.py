"""The 8-bit floating-point operators against plain ones in 64 bits (fp8_ref.py), through the public calls.

Rows into 8 bits are exact: the scale is a power of two, so every value has one nearest e4m3 number.  Products have the
bound that fp8_ref.product derives.  silu(gate) * up is formed in f32: exp is off by at most 2^-23 of it, the sum, the quotient
and the product round once each, so h is off by at most 5 * 2^-24 of it, and the number chosen is as near to h as the
nearest is but for that.
"""
import numpy as np
import pytest
import torch

from . import fp8_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ACTS = [F32, F16, BF16]


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import lloom_amd

    lloom_amd.lib()
    return lloom_amd


def normal(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def f64(t):
    return t.detach().cpu().double().numpy()


def same_rows(q, s, x):
    want, ws = R.quantize(f64(x).reshape(-1, x.shape[-1]))
    got = q.cpu().view(torch.uint8).numpy().reshape(want.shape)
    nan = (want & 127) == 127
    assert np.array_equal(f64(s), ws)
    assert np.array_equal(got[~nan], want[~nan]) and np.array_equal((got & 127) == 127, nan)


# ------------------------------------------------------------------- rows --

@pytest.mark.parametrize("dtype", ACTS)
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 128), (3, 144), (5, 2048), (17, 528), (67, 1376), (2049, 2064), (4100, 1024)])
def test_rows(L, rows, k, dtype):
    x = normal(rows + k, rows, k, std=3.0)
    x[0, :16] = torch.tensor([0.0, -0.0, 1e-30, 448.0, -448.0, 464.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 0.0625, 17.0,
                              19.0, 21.0, -23.0, 30000.0, 1e-7])
    x = x.to(dtype)
    same_rows(*L.fp8_quantize(x.cuda()), x)


def test_every_boundary_of_a_scale(L):
    """Largest values at, just under and just over 448 * 2^e for every e that f32 has, among ties and subnormals."""
    rows = []
    for e in range(-149 - 8, 128 - 8):
        top = 448.0 * 2.0 ** e
        for t in (np.float32(top), np.nextafter(np.float32(top), np.float32(0)), np.nextafter(np.float32(top), np.float32(np.inf))):
            if np.isfinite(t):
                rows.append(np.concatenate([[t], t * np.linspace(-1, 1, 127)]).astype(np.float32))
    x = torch.from_numpy(np.stack(rows))
    same_rows(*L.fp8_quantize(x.cuda()), x)


def test_every_half_and_tie(L):
    """Every finite f16, 128 at a time: all ties between e4m3 numbers are among them."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(F16)
    x = x[torch.isfinite(x)][: 63488 // 128 * 128].reshape(-1, 128)
    same_rows(*L.fp8_quantize(x.cuda()), x)


@pytest.mark.parametrize("dtype", ACTS)
def test_rows_that_are_no_numbers(L, dtype):
    x = normal(5, 6, 256)
    x[0] = 0
    x[1, 7], x[1, 200] = float("nan"), float("inf")
    x[2] = float("-inf")
    x[3, :128] = float("nan")
    x[4, 128:] = -0.0
    x = x.to(dtype)
    q, s = L.fp8_quantize(x.cuda())
    same_rows(q, s, x)
    assert f64(s)[0].tolist() == [1.0, 1.0] and f64(s)[2].tolist() == [1.0, 1.0]


def test_layouts(L):
    base = normal(6, 40, 1024, dtype=F16).cuda()
    for x in (base[:, 256:768], base[::3, :512], base[1:, 8:136], base.t()[:48, :32], base[:, 4:132], base[:0]):
        q, s = L.fp8_quantize(x)
        assert q.shape == x.shape and s.shape == (x.shape[0], -(-x.shape[1] // 128))
        same_rows(q, s, x)
    x = base.reshape(4, 10, 1024)
    q, s = L.fp8_quantize(x)
    assert q.shape == x.shape
    same_rows(q, s, x)


# -------------------------------------------------------------------- gate --

@pytest.mark.parametrize("dtype", ACTS)
@pytest.mark.parametrize("rows,k", [(1, 16), (37, 1376), (2100, 2048)])
def test_gate(L, rows, k, dtype):
    both = normal(rows, rows, 2 * k, std=4.0, dtype=dtype)
    both[0, :4] = torch.tensor([100.0, -100.0, 0.0, -88.0])
    dev = both.cuda()
    q, s = L.fp8_silu_mul(dev[:, :k], dev[:, k:])
    g, u = f64(both[:, :k]), f64(both[:, k:])
    with np.errstate(over="ignore"):
        h = g / (1 + np.exp(-g)) * u
    off = 5 * 2.0 ** -24 * np.abs(h) + 2.0 ** -126
    got, gs = R.values(q), f64(s)
    # a scale may differ where the block's largest is within `off` of a boundary
    kb = gs.shape[1]
    pad = np.zeros((rows, kb * 128))
    pad[:, :k] = np.abs(h)
    top = pad.reshape(rows, kb, 128).max(2)
    low, high = R.scale(top * (1 - 2.0 ** -21)), R.scale(top * (1 + 2.0 ** -21))
    assert np.all((gs == low) | (gs == high))
    wide = np.repeat(gs, 128, 1)[:, :k]
    near = R.TABLE[R.nearest(np.clip(h / wide, -448, 448))]
    assert np.all(np.abs(got * wide - h) <= np.abs(near * wide - h) + 2 * off)


def test_gate_is_the_formula_in_f32(L):
    """The same numbers as the formula's steps in f32 elementwise operations give."""
    g, u = normal(8, 600, 2048).cuda() * 3, normal(9, 600, 2048).cuda()
    q, s = L.fp8_silu_mul(g, u)
    q2, s2 = L.fp8_quantize(g / (1.0 + torch.exp(-g)) * u)
    assert torch.equal(s, s2) and (q.view(torch.uint8) != q2.view(torch.uint8)).float().mean().item() < 1e-4


def test_gate_near_the_end_of_the_exponential(L):
    """Gates of -88.5 to -60, sixteen neighbours of one value, with an `up` that brings them to the middle of f32: the
    formula's few roundings (as in test_gate) and e4m3's."""
    g = torch.linspace(-88.5, -60, 64 * 512).reshape(64, 512, 1).expand(64, 512, 16).reshape(64, 8192).contiguous()
    u = torch.full_like(g, 2.0 ** 100)
    q, s = L.fp8_silu_mul(g.cuda(), u.cuda())
    h = f64(g) / (1 + np.exp(-f64(g))) * 2.0 ** 100
    got = R.values(q) * np.repeat(f64(s), 128, 1)
    # eight values of 16 a block, at most e^.007 apart: all in one or two steps of e4m3, half a step of at most 2^-3 off
    assert np.all(np.abs(got - h) <= (2.0 ** -4 + 2.0 ** -20) * np.abs(h))


# ----------------------------------------------------------------- weights --

@pytest.mark.parametrize("dtype", ACTS)
@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 272), (3, 200, 400), (2, 16, 2048)])
def test_weights(L, shape, dtype):
    w = normal(sum(shape), *shape, dtype=dtype, std=0.02)
    q, s = L.fp8_quantize_weight(w.cuda())
    n, k = shape[-2:]
    w3, q3 = f64(w).reshape(-1, n, k), q.cpu().view(torch.uint8).numpy().reshape(-1, n, k)
    s3 = f64(s).reshape(-1, -(-n // 128), -(-k // 128))
    for e in range(len(w3)):
        pad = np.zeros((s3.shape[1] * 128, s3.shape[2] * 128))
        pad[:n, :k] = np.abs(w3[e])
        want = R.scale(pad.reshape(s3.shape[1], 128, s3.shape[2], 128).max((1, 3)))
        assert np.array_equal(s3[e], want)
        assert np.array_equal(q3[e], R.nearest(w3[e] / R.spread(want, n, k)))


# ---------------------------------------------------------------- products --

def weights(seed, *shape):
    """e4m3 weights of all sizes and f32 scales of any value."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(*shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128), generator=g) * 0.01 + 1e-4
    return q, s


def halves(dtype):
    return dtype is not F32


def check_product(y, x, xs, w, ws):
    """y against x (as given to the call) times w."""
    if xs is None:
        q, sx = R.quantize(f64(x).reshape(-1, x.shape[-1]))
        q = R.TABLE[q]
    else:
        q, sx = R.values(x), f64(xs)
    want, off = R.product(q, sx, R.values(w), f64(ws), y.dtype, halves(y.dtype))
    got = f64(y).reshape(want.shape)
    assert np.all(np.abs(got - want) <= off), np.max(np.abs(got - want) / off)


SIZES = [(1, 16, 16), (1, 6152, 912), (1, 80, 8208), (4, 16400, 272), (12, 4104, 2064), (1, 64, 128), (2, 24, 144),
         (5, 130, 272), (16, 128, 2048), (17, 257, 1040), (33, 96, 96), (64, 384, 640),
         (65, 200, 1376), (129, 127, 512), (255, 264, 768), (300, 520, 256), (1030, 1000, 400),
         (2100, 264, 144), (2049, 300, 912)]


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("m,n,k", [(2100, 264, 16), (2100, 264, 272), (540, 1000, 1152), (1100, 1000, 16), (1100, 1000, 528),
                                   (700, 1500, 2064), (1030, 2900, 4112), (520, 4200, 2064), (3400, 3101, 144),
                                   (40, 4103, 272), (70, 9001, 144)])
def test_matmul_of_an_odd_number_of_blocks(L, m, n, k, out):
    w, ws = weights(n + k, n, k)
    q, sx = (t.cpu() for t in L.fp8_quantize(normal(m, m, k).cuda()))
    ws[0, -1] = 3e38  # past the end of the rows nothing may meet it
    sx[0, -1] = 3e38
    sx, ws = sx * 2.0 ** -64, ws * 2.0 ** -64
    y = L.fp8_matmul(q.cuda(), w.cuda(), ws.cuda(), x_scales=sx.cuda(), out_dtype=out).cpu()
    check_product(y[1:], q[1:], sx[1:], w, ws)
    check_product(y[:1, 128:], q[:1], sx[:1], w[128:], ws[1:])
    # where the two scales meet (2.6e38, in f32's range) sums of 1.4 and more are past its largest, 3.4e38
    d = R.values(q)[0, -((k - 1) % 128 + 1):] @ R.values(w)[:128, -((k - 1) % 128 + 1):].T
    assert np.array_equal(f64(y)[0, :128][np.abs(d) > 1.4], np.copysign(np.inf, d[np.abs(d) > 1.4]))


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(L, m, n, k, out):
    w, ws = weights(n + k, n, k)
    x = normal(m, m, k, dtype=out)
    check_product(L.fp8_matmul(x.cuda(), w.cuda(), ws.cuda()), x, None, w, ws)
    q, sx = (t.cpu() for t in L.fp8_quantize(x.cuda()))
    sx = sx * torch.rand(sx.shape, generator=torch.Generator().manual_seed(m))  # scales of any value
    for scales in (sx, sx.t().contiguous().t()):
        y = L.fp8_matmul(q.cuda(), w.cuda(), ws.cuda(), x_scales=scales.cuda(), out_dtype=out)
        check_product(y, q, sx, w, ws)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("out", ACTS)
def test_types_in_and_out(L, act, out):
    w, ws = weights(3, 200, 400)
    for m in (1, 20, 200):
        x = normal(m, m, 400, dtype=act)
        y = L.fp8_matmul(x.cuda(), w.cuda(), ws.cuda(), out_dtype=out)
        assert y.dtype is out
        check_product(y, x, None, w, ws)


def ragged(counts, extra, seed):
    """Starts of groups of these sizes with `extra` rows of none behind, and an order of the rows."""
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1]) + extra
    return torch.tensor(starts, dtype=torch.int32), rows, torch.randperm(rows, generator=torch.Generator().manual_seed(seed))


GROUPS = [([3], 0), ([0, 1, 16, 17, 0, 5], 0), ([15, 16, 17, 31, 32, 33, 0, 64, 65, 1], 3), ([127, 128, 129, 0, 255, 257], 1),
          ([0, 0, 0], 5), ([1] * 70, 0), ([0] * 130 + [9] + [0] * 60, 2), ([600, 1], 0),
          ([1000, 0, 3, 1200, 257], 9), ([1, 0, 2, 1, 0, 4], 2), ([3] * 600, 7)]


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("counts,extra", GROUPS)
def test_grouped(L, counts, extra, out):
    n, k, E = 136, 272, len(counts)
    starts, rows, order = ragged(counts, extra, E)
    w, ws = weights(E, E, n, k)
    tokens = max(1, rows // 2)
    x = normal(rows, tokens, k, dtype=out)
    gather = (order % tokens).int()
    y = L.fp8_grouped_matmul(x.cuda(), w.cuda(), ws.cuda(), starts.cuda(), gather=gather.cuda(), scatter=order.int().cuda())
    assert y.shape == (rows, n)
    q, sx = (t.cpu() for t in L.fp8_quantize(x.cuda()))
    y2 = L.fp8_grouped_matmul(q[gather.long()].cuda(), w.cuda(), ws.cuda(), starts.cuda(), x_scales=sx[gather.long()].cuda(),
                              out_dtype=out)
    y = y.cpu()
    for e, c in enumerate(counts):
        i = torch.arange(int(starts[e]), int(starts[e]) + c)
        if c:
            check_product(y[order[i]], x[gather[i].long()], None, w[e], ws[e])
            check_product(y2[i.cuda()], x[gather[i].long()], None, w[e], ws[e])
    i = torch.arange(int(starts[-1]), rows)
    assert not y[order[i]].any() and not y2[i.cuda()].any()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("counts", [[16], [13], [9, 7], [5, 0, 10], [17], [30, 3], [40, 1, 0]])
def test_few_experts_of_few_rows(L, counts, act):
    """Rows of every type around the 16 that workgroups bring into 8 bits themselves, for fewer experts than that counts."""
    starts, rows, order = ragged(counts, 0, 3)
    w, ws = weights(rows, len(counts), 80, 400)
    x = normal(rows, rows, 400, dtype=act)
    y = L.fp8_grouped_matmul(x.cuda(), w.cuda(), ws.cuda(), starts.cuda(), gather=order.int().cuda())
    for e, c in enumerate(counts):
        i = slice(int(starts[e]), int(starts[e]) + c)
        if c:
            check_product(y[i], x[order[i]], None, w[e], ws[e])


# -------------------------------------------------------------------- plan --

def plan_of(ids, experts):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    starts = torch.searchsorted(key[order], torch.arange(experts + 1))
    return starts, order, order // ids.shape[1]


@pytest.mark.parametrize("tokens,topk,experts", [(1, 1, 1), (1, 8, 64), (3, 2, 5), (32, 8, 128), (257, 4, 8), (2048, 1, 3),
                                                 (1000, 7, 4096), (8192, 8, 128), (33333, 3, 9)])
def test_plan(L, tokens, topk, experts):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1 if tokens > 1 else 0, experts, (tokens, topk), generator=g, dtype=torch.int32)
    p = L.expert_plan(ids.cuda(), experts)
    for got, want in zip(p, plan_of(ids, experts)):
        assert got.dtype is torch.int32 and torch.equal(got.cpu().long(), want)
    L.paged_check()


@pytest.mark.parametrize("tokens,hot", [(3000, 1.0), (40000, 1.0), (40000, 0.9), (40000, 0.5), (200000, 0.2)])
def test_plan_of_one_liked_expert(L, tokens, hot):
    """More planes of one expert than a wave lists at once, in all waves or in some, and many of none."""
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-2, 7, (tokens, 2), generator=g, dtype=torch.int32)
    ids[torch.rand(tokens, 2, generator=g) < hot] = 3
    ids[tokens // 3: tokens // 2] = -1
    p = L.expert_plan(ids.cuda(), 7)
    for got, want in zip(p, plan_of(ids, 7)):
        assert torch.equal(got.cpu().long(), want)
    L.paged_check()


def test_plan_reports_ids_past_the_last_expert(L):
    L.paged_check()
    ids = torch.tensor([[0, 7], [3, -5], [2 ** 31 - 1, 1]], dtype=torch.int32)
    p = L.expert_plan(ids.cuda(), 4)
    for got, want in zip(p, plan_of(ids, 4)):
        assert torch.equal(got.cpu().long(), want)
    with pytest.raises(L.LloomHipError) as e:
        L.paged_check()
    assert e.value.name == "EEXPERT"
    L.paged_check()


def test_no_tokens(L):
    p = L.expert_plan(torch.zeros(0, 4, dtype=torch.int32, device="cuda"), 3)
    assert p.starts.tolist() == [0, 0, 0, 0] and p.planes.numel() == p.tokens.numel() == 0
    w, ws = (t.cuda() for t in weights(1, 3, 32, 64))
    assert L.fp8_matmul(torch.empty(0, 64, device="cuda"), w[0], ws[0]).shape == (0, 32)
    y = L.fp8_grouped_matmul(torch.empty(0, 64, device="cuda"), w, ws, p.starts, gather=p.tokens)
    assert y.shape == (0, 32)
