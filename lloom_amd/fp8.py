"""Products with 8-bit floating-point weights (e4m3, a scale for each block of 128 x 128), dense and grouped by expert (the C
ABI's lloom_hip_fp8_* and lloom_hip_expert_plan), beside the packed integer ones of quantized.py.

A weight is a pair of tensors as checkpoints hold them: e4m3 [.., n, k] (torch.float8_e4m3fn) and f32 scales
[.., ceil(n / 128), ceil(k / 128)].  Activations are f32, f16 or bf16 rows, which a product brings into 8 bits itself, or e4m3
rows with a scale for each 128 values (fp8_quantize, fp8_silu_mul), where several products share them.  k is a multiple of 16.

An expert layer of a step is

    plan = expert_plan(ids, experts)                                                          # ids [tokens, topk]
    h = fp8_grouped_matmul(x, w_up, s_up, plan.starts, gather=plan.tokens)                    # [planes, 2 * inner]
    q, s = fp8_silu_mul(h[:, :inner], h[:, inner:])
    y = fp8_grouped_matmul(q, w_down, s_down, plan.starts, x_scales=s, scatter=plan.planes, out_dtype=x.dtype)

with y [tokens * topk, n] in the order of ids, as QTensor.indexed_moe_forward has it.  A product that brings x into 8 bits in a
launch before its own does so in the workspace of the GPU's context, which serves one stream at a time: calls on another stream
wait for them first, or take e4m3 x (fp8_quantize's).  Nothing here waits for the GPU: what
only the GPU can see (an id, a start or a row out of range) is left out of the result and raised by the next paged_check()
as EEXPERT.
"""
import ctypes
from typing import NamedTuple

import torch

from .lib import LloomHipError, check, lib
from .quantized import MMA_F16, _ctx, _ctxs, _stream_of  # noqa: F401

E4M3 = torch.float8_e4m3fn
_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30, E4M3: 100}
BLOCK = 128
MMA_FP8 = 3
MAX_EXPERTS = 4096  # the library refuses more


class ExpertPlan(NamedTuple):
    """Planes (token * topk + slot) in the order of their experts, int32 on the GPU."""
    starts: torch.Tensor  # [experts + 1]: the first place of each expert's planes; the last: of those that have no expert
    planes: torch.Tensor  # [tokens * topk]
    tokens: torch.Tensor  # [tokens * topk]: the planes' tokens


# The host's part of a call is most of a small one's time, so what is common is looked at first and once; what is not as
# common expects it goes to _rows and the messages.

def _gpu(t, what):
    """The context of the GPU that t is on."""
    i = t.get_device()
    if i < 0:
        raise LloomHipError(1, f"{what}: a tensor on {t.device} is not on a HIP device")
    return _ctxs.get(i) or _ctx(i)


def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _rows(x, what, e4m3=False):
    """x as rows [rows, k] that the kernels read, their number, k, and how far apart they are: dense in k, 16-byte aligned;
    another layout is copied."""
    d = x.dtype
    if d not in _IDS or (d is E4M3) != e4m3:
        raise LloomHipError(2, f"{what}: {d} is not " + ("e4m3" if e4m3 else "an activation dtype (f32, f16 or bf16)"))
    shape = x.shape
    if len(shape) != 2:
        if not shape:
            raise LloomHipError(3, f"{what}: a tensor of no dimension is no rows")
        x = x.reshape(-1, shape[-1]) if x.numel() else x.new_empty((shape[:-1].numel(), shape[-1]))
        shape = x.shape
    rows, k = shape
    if k == 0 or k % 16:
        raise LloomHipError(3, f"{what}: rows of {k} values: k must be a multiple of 16")
    if x.is_contiguous() and not x.data_ptr() % 16:
        return x, rows, k, k
    s0, s1 = x.stride()
    if rows and (s1 != 1 or s0 < k or s0 * x.element_size() % 16 or x.data_ptr() % 16):
        return x.clone(memory_format=torch.contiguous_format), rows, k, k
    return x, rows, k, max(s0, k)


def _new_rows(like, rows, k):
    """e4m3 of a tensor's shape, and the rows' scales, block by block in memory."""
    q = torch.empty_like(like, dtype=E4M3, memory_format=torch.contiguous_format)
    return q, torch.empty_strided((rows, (k + 127) // 128), (1, rows), dtype=torch.float32, device=like.device)


def fp8_quantize(x):
    """Rows of x [.., k] (f32, f16 or bf16) as e4m3 [.., k] and f32 scales [rows, ceil(k / 128)]: a block's scale is 2^e with
    the least e >= -126 for which its largest finite value is at most 448 * 2^e (1 for zeros), its values the nearest e4m3
    numbers of x / scale (ties to even; infinities and NaN give NaN)."""
    ctx = _gpu(x, "fp8_quantize")
    r, rows, k, stride = _rows(x, "fp8_quantize")
    q, s = _new_rows(x, rows, k)
    rc = lib().lloom_hip_fp8_quantize(ctx, r.data_ptr(), _IDS[r.dtype], stride, rows, k, q.data_ptr(), s.data_ptr(), rows,
                                      _stream_of(x.get_device()))
    if rc:
        check(rc)
    return q, s


def fp8_silu_mul(gate, up):
    """fp8_quantize of silu(gate) * up = gate / (1 + exp(-gate)) * up, formed in f32; gate and up [.., k] of one dtype (two
    halves of one product's rows are read where they are)."""
    ctx = _gpu(gate, "fp8_silu_mul")
    i = gate.get_device()
    if gate.dtype is not up.dtype or gate.shape != up.shape or up.get_device() != i:
        raise LloomHipError(3, f"fp8_silu_mul: gate {tuple(gate.shape)} {gate.dtype} on {gate.device} and up "
                               f"{tuple(up.shape)} {up.dtype} on {up.device} differ")
    g, rows, k, gs = _rows(gate, "fp8_silu_mul")
    u, _, _, us = _rows(up, "fp8_silu_mul")
    q, s = _new_rows(gate, rows, k)
    rc = lib().lloom_hip_fp8_silu_mul(ctx, g.data_ptr(), gs, u.data_ptr(), us, _IDS[g.dtype], rows, k, q.data_ptr(),
                                      s.data_ptr(), rows, _stream_of(i))
    if rc:
        check(rc)
    return q, s


def fp8_quantize_weight(w):
    """A weight [n, k] or weights [experts, n, k] (f32, f16 or bf16) as e4m3 of the same shape and f32 scales
    [.., ceil(n / 128), ceil(k / 128)], chosen as fp8_quantize does for blocks of 128 x 128."""
    ctx = _gpu(w, "fp8_quantize_weight")
    if w.dtype not in _IDS or w.dtype is E4M3:
        raise LloomHipError(2, f"fp8_quantize_weight: {w.dtype} is not f32, f16 or bf16")
    if w.dim() not in (2, 3) or w.numel() == 0:
        raise LloomHipError(3, f"fp8_quantize_weight: {tuple(w.shape)} is not [n, k] or [experts, n, k]")
    w = w.contiguous()
    if w.data_ptr() % 16:
        w = w.clone()
    experts = w.shape[0] if w.dim() == 3 else 1
    n, k = w.shape[-2:]
    q = torch.empty(w.shape, dtype=E4M3, device=w.device)
    s = torch.empty(w.shape[:-2] + (_blocks(n), _blocks(k)), dtype=torch.float32, device=w.device)
    check(lib().lloom_hip_fp8_quantize_weight(ctx, w.data_ptr(), _IDS[w.dtype], experts, n, k, q.data_ptr(), s.data_ptr(),
                                              _stream_of(w.get_device())))
    return q, s


def _weight(w, s, dim, what):
    """Refuses what is no e4m3 weight of `dim` dimensions with the scales of its blocks."""
    shape, blocks = w.shape, s.shape
    if w.dtype is not E4M3 or s.dtype is not torch.float32:
        raise LloomHipError(2, f"{what}: a weight of {w.dtype} with scales of {s.dtype} is not e4m3 with f32 scales")
    if (len(shape) != dim or len(blocks) != dim or blocks[-2] != (shape[-2] + 127) // 128
            or blocks[-1] != (shape[-1] + 127) // 128 or blocks[0] != (shape[0] if dim == 3 else blocks[0])
            or not w.is_contiguous() or not s.is_contiguous() or s.get_device() != w.get_device()):
        raise LloomHipError(3, f"{what}: a weight {tuple(shape)} on {w.device} with scales {tuple(blocks)} on {s.device} is "
                               f"no contiguous weight of {dim} dimensions with contiguous scales of its blocks of 128 x 128")
    return shape


def _x(x, x_scales, i, k, what):
    """Rows of x, their number and how far apart they are, the address of their scales (0: none) and how far apart those
    are, by row and by block."""
    r, rows, xk, stride = _rows(x, what, x_scales is not None)
    if xk != k or r.get_device() != i:
        raise LloomHipError(3, f"{what}: x {tuple(x.shape)} on {x.device} does not fit a weight of k {k} on GPU {i}")
    if x_scales is None:
        return r, rows, stride, 0, 0, 0
    if x_scales.dtype is not torch.float32 or x_scales.shape != (rows, (k + 127) // 128) or x_scales.get_device() != i:
        raise LloomHipError(3, f"{what}: scales {tuple(x_scales.shape)} {x_scales.dtype} on {x_scales.device} are not f32 "
                               f"[{rows}, {_blocks(k)}] on GPU {i}")
    s0, s1 = x_scales.stride()
    return r, rows, stride, x_scales.data_ptr(), s0, s1


def _out_dtype(x, x_scales, out_dtype, out, what):
    d = out_dtype or (x.dtype if x_scales is None else torch.float32 if out is None else out.dtype)
    if d not in _IDS or d is E4M3:
        raise LloomHipError(2, f"{what}: {d} is not an output dtype (f32, f16 or bf16)")
    return d


def _new(like, dtype, rows, n):
    return like.new_empty((rows, n)) if like.dtype is dtype else torch.empty((rows, n), dtype=dtype, device=like.device)


def _check_out(out, shape, dtype, i, what):
    if out.dtype is not dtype or out.shape != shape or not out.is_contiguous() or out.get_device() != i:
        raise LloomHipError(3, f"{what}: out {tuple(out.shape)} {out.dtype} on {out.device} does not fit the contiguous "
                               f"{dtype} output {tuple(shape)} on GPU {i}")


def fp8_matmul(x, weight, weight_scales, x_scales=None, out_dtype=None, out=None):
    """x . W^T for a weight e4m3 [n, k] with f32 scales [ceil(n / 128), ceil(k / 128)]; x [.., k] f32, f16 or bf16 (brought
    into 8 bits as fp8_quantize does), or e4m3 with x_scales [rows, ceil(k / 128)].  The result [.., n] is of out_dtype (x's
    own by default, f32 for e4m3 x): exact products, sums in f32 (but for set_fp8_mma), rounded once.  `out`
    shares no memory with what the call reads."""
    ctx = _gpu(weight, "fp8_matmul")
    i = weight.get_device()
    n, k = _weight(weight, weight_scales, 2, "fp8_matmul")
    r, rows, stride, xs, s0, s1 = _x(x, x_scales, i, k, "fp8_matmul")
    d = _out_dtype(x, x_scales, out_dtype, out, "fp8_matmul")
    if out is None:
        out = _new(r, d, rows, n)
        if len(x.shape) != 2:
            out = out.view(x.shape[:-1] + (n,))
    else:
        _check_out(out, x.shape[:-1] + (n,), d, i, "fp8_matmul")
    rc = lib().lloom_hip_fp8_matmul(ctx, weight.data_ptr(), weight_scales.data_ptr(), n, k, r.data_ptr(), _IDS[r.dtype],
                                    stride, xs, s0, s1, rows, out.data_ptr(), _IDS[d], _stream_of(i))
    if rc:
        check(rc)
    return out


def expert_plan(ids, experts):
    """The order of a step's planes by expert: ids [tokens, topk] (int32), each in [0, experts).  Planes of one expert keep
    their order.  A negative id is a plane of no expert (a padded batch); one past the last expert is too, and paged_check()
    raises.  Such planes come last, and the products' rows for them are zero."""
    ctx = _gpu(ids, "expert_plan")
    if ids.dtype is not torch.int32 or ids.dim() != 2:
        raise LloomHipError(2, f"expert_plan: ids {tuple(ids.shape)} {ids.dtype} are not int32 [tokens, topk]")
    if not ids.is_contiguous():
        ids = ids.contiguous()
    tokens, topk = ids.shape
    p = tokens * topk
    buf = ids.new_empty(2 * p + min(max(experts, 0), MAX_EXPERTS) + 1)
    base = buf.data_ptr()
    rc = lib().lloom_hip_expert_plan(ctx, ids.data_ptr(), tokens, topk, experts, base + 8 * p, base, base + 4 * p,
                                     _stream_of(ids.get_device()))
    if rc:
        check(rc)
    planes, of, starts = buf.split((p, p, experts + 1))
    return ExpertPlan(starts, planes, of)


def _index(t, i, what):
    if t is None and what != "starts":
        return 0
    if not isinstance(t, torch.Tensor):
        raise LloomHipError(1, f"fp8_grouped_matmul: {what} is a {type(t).__name__}, no tensor")
    if t.dtype is not torch.int32 or t.dim() != 1 or t.get_device() != i or not t.is_contiguous():
        raise LloomHipError(2, f"fp8_grouped_matmul: {what} {tuple(t.shape)} {t.dtype} on {t.device} is not a dense int32 "
                               f"tensor of one dimension on GPU {i}")
    return t.data_ptr()


def fp8_grouped_matmul(x, weight, weight_scales, starts, x_scales=None, gather=None, scatter=None, out_dtype=None, out=None):
    """Products grouped by expert, ragged: weights e4m3 [experts, n, k] with scales [experts, ceil(n / 128), ceil(k / 128)];
    row i with starts[e] <= i < starts[e + 1] (int32 [experts + 1], from 0, not falling) is x[gather[i]] (int32; None: x[i])
    times weight e, and is stored at out[scatter[i]] (int32, no two alike; None: out[i]).  Rows of no expert are zero.  x,
    x_scales and the sums as in fp8_matmul; the result [rows, n] has a row for each of gather, scatter or x, in that order of
    preference.  With scatter, `out` may have more rows; those that scatter does not name are left as they are."""
    what = "fp8_grouped_matmul"
    ctx = _gpu(weight, what)
    i = weight.get_device()
    experts, n, k = _weight(weight, weight_scales, 3, what)
    r, x_rows, stride, xs, s0, s1 = _x(x, x_scales, i, k, what)
    g, c, st = _index(gather, i, "gather"), _index(scatter, i, "scatter"), _index(starts, i, "starts")
    rows = x_rows if gather is None and scatter is None else (scatter if gather is None else gather).shape[0]
    if (starts.shape[0] != experts + 1 or (gather is None and x_rows < rows)
            or (scatter is not None and scatter.shape[0] != rows)):
        raise LloomHipError(3, f"{what}: {starts.shape[0]} starts of {experts} experts, {rows} rows of {x_rows}"
                               + ("" if scatter is None else f" to {scatter.shape[0]} places"))
    d = _out_dtype(x, x_scales, out_dtype, out, what)
    y_rows = rows
    if out is None:
        out = _new(r, d, rows, n)
    else:
        if scatter is not None and out.dim() == 2:
            y_rows = max(rows, out.shape[0])
        _check_out(out, (y_rows, n), d, i, what)
    rc = lib().lloom_hip_fp8_grouped_matmul(ctx, weight.data_ptr(), weight_scales.data_ptr(), experts, n, k, r.data_ptr(),
                                            _IDS[r.dtype], stride, xs, s0, s1, x_rows, st, g, c, rows, out.data_ptr(),
                                            _IDS[d], y_rows, _stream_of(i))
    if rc:
        check(rc)
    return out


def set_fp8_mma(mode, device=0):
    """Matrix-core family of the products of many rows into f16 and bf16: MMA_F16 (the default: the numbers as halves, exact
    products, f32 sums, as into f32 and of few rows always) or MMA_FP8 (the 8-bit instructions, at twice the rate, which cut
    off what is under 2^-13 of the largest of eight neighbours' products: 1.5e-5 of the result in the 2-norm for normal
    values, and all that is left where large neighbours cancel)."""
    check(lib().lloom_hip_ctx_set_fp8_mma(_ctx(device), mode))


def fp8_workspace_bytes(dtype, rows, k, x_rows=None, experts=0):
    """The workspace a product of `rows` rows takes (reserve_workspace it before a capture): x of dtype [x_rows, k], as many
    as rows by default; experts: 0 for fp8_matmul."""
    if dtype not in _IDS:
        raise LloomHipError(2, f"fp8_workspace_bytes: {dtype} is not f32, f16, bf16 or e4m3")
    out = ctypes.c_size_t()
    check(lib().lloom_hip_fp8_workspace_bytes(_IDS[dtype], rows, rows if x_rows is None else x_rows, experts, k,
                                              ctypes.byref(out)))
    return out.value
