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

with y [tokens * topk, n] in the order of ids, as QTensor.indexed_moe_forward has it.  Nothing here waits for the GPU: what
only the GPU can see (an id, a start or a row out of range) is left out of the result and raised by the next paged_check()
as EEXPERT.
"""
import ctypes
from typing import NamedTuple

import torch

from .lib import LloomHipError, check, lib
from .quantized import _ctx, _ctxs, _stream_of

E4M3 = torch.float8_e4m3fn
_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30, E4M3: 100}
BLOCK = 128


class ExpertPlan(NamedTuple):
    """Planes (token * topk + slot) in the order of their experts, int32 on the GPU."""
    starts: torch.Tensor  # [experts + 1]: the first place of each expert's planes; the last: of those that have no expert
    planes: torch.Tensor  # [tokens * topk]
    tokens: torch.Tensor  # [tokens * topk]: the planes' tokens


def _gpu(t, what):
    """The GPU that t is on, and the handle of its context."""
    i = t.get_device()
    if i < 0:
        raise LloomHipError(1, f"{what}: a tensor on {t.device} is not on a HIP device")
    return i, _ctxs.get(i) or _ctx(i)


def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _rows(x, what, e4m3=False):
    """x as rows [rows, k] that the kernels read: dense in k, 16-byte aligned; another layout is copied."""
    d = x.dtype
    if d not in _IDS or (d is E4M3) != e4m3:
        raise LloomHipError(2, f"{what}: {d} is not " + ("e4m3" if e4m3 else "an activation dtype (f32, f16 or bf16)"))
    if x.dim() != 2:
        if x.dim() == 0:
            raise LloomHipError(3, f"{what}: a tensor of no dimension is no rows")
        x = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty((x.shape[:-1].numel(), x.shape[-1]))
    k = x.shape[1]
    if k == 0 or k % 16:
        raise LloomHipError(3, f"{what}: rows of {k} values: k must be a multiple of 16")
    s0, s1 = x.stride()
    if (s1 != 1 or s0 < k or s0 * x.element_size() % 16 or x.data_ptr() % 16) and x.numel():
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _stride(x):
    return max(x.stride(0), x.shape[1])


def _new_rows(x, rows, k, shape):
    """e4m3 rows and their scales, block by block in memory."""
    q = torch.empty(shape, dtype=E4M3, device=x.device)
    return q, torch.empty((_blocks(k), rows), dtype=torch.float32, device=x.device)


def fp8_quantize(x):
    """Rows of x [.., k] (f32, f16 or bf16) as e4m3 [.., k] and f32 scales [rows, ceil(k / 128)]: a block's scale is 2^e with
    the least e >= -126 for which its largest finite value is at most 448 * 2^e (1 for zeros), its values the nearest e4m3
    numbers of x / scale (ties to even; infinities and NaN give NaN)."""
    i, ctx = _gpu(x, "fp8_quantize")
    r = _rows(x, "fp8_quantize")
    rows, k = r.shape
    q, s = _new_rows(x, rows, k, x.shape)
    check(lib().lloom_hip_fp8_quantize(ctx, r.data_ptr(), _IDS[r.dtype], _stride(r), rows, k, q.data_ptr(), s.data_ptr(),
                                       rows, _stream_of(i)))
    return q, s.t()


def fp8_silu_mul(gate, up):
    """fp8_quantize of silu(gate) * up = gate / (1 + exp(-gate)) * up, formed in f32; gate and up [.., k] of one dtype (two
    halves of one product's rows are read where they are)."""
    i, ctx = _gpu(gate, "fp8_silu_mul")
    if gate.dtype is not up.dtype or gate.shape != up.shape or up.get_device() != i:
        raise LloomHipError(3, f"fp8_silu_mul: gate {tuple(gate.shape)} {gate.dtype} on {gate.device} and up "
                               f"{tuple(up.shape)} {up.dtype} on {up.device} differ")
    g, u = _rows(gate, "fp8_silu_mul"), _rows(up, "fp8_silu_mul")
    rows, k = g.shape
    q, s = _new_rows(gate, rows, k, gate.shape)
    check(lib().lloom_hip_fp8_silu_mul(ctx, g.data_ptr(), _stride(g), u.data_ptr(), _stride(u), _IDS[g.dtype], rows, k,
                                       q.data_ptr(), s.data_ptr(), rows, _stream_of(i)))
    return q, s.t()


def fp8_quantize_weight(w):
    """A weight [n, k] or weights [experts, n, k] (f32, f16 or bf16) as e4m3 of the same shape and f32 scales
    [.., ceil(n / 128), ceil(k / 128)], chosen as fp8_quantize does for blocks of 128 x 128."""
    i, ctx = _gpu(w, "fp8_quantize_weight")
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
                                              _stream_of(i)))
    return q, s


def _weight(w, s, dim, i, what):
    """n and k of an e4m3 weight of `dim` dimensions with its scales."""
    if w.dtype is not E4M3 or s.dtype is not torch.float32:
        raise LloomHipError(2, f"{what}: a weight of {w.dtype} with scales of {s.dtype} is not e4m3 with f32 scales")
    shape = w.shape
    if (len(shape) != dim or s.shape != shape[:-2] + (_blocks(shape[-2]), _blocks(shape[-1])) or not w.is_contiguous()
            or not s.is_contiguous() or w.get_device() != i or s.get_device() != i):
        raise LloomHipError(3, f"{what}: a weight {tuple(shape)} on {w.device} with scales {tuple(s.shape)} on {s.device} is "
                               f"no contiguous weight of {dim} dimensions on GPU {i} with scales of its blocks of 128 x 128")
    return shape[-2], shape[-1]


def _x(x, x_scales, i, k, what):
    """Rows of x, the address of their scales (0: none) and how far apart those are."""
    r = _rows(x, what, x_scales is not None)
    if r.shape[1] != k or r.get_device() != i:
        raise LloomHipError(3, f"{what}: x {tuple(x.shape)} on {x.device} does not fit a weight of k {k} on GPU {i}")
    if x_scales is None:
        return r, 0, 0, 0
    if x_scales.dtype is not torch.float32 or x_scales.shape != (r.shape[0], _blocks(k)) or x_scales.get_device() != i:
        raise LloomHipError(3, f"{what}: scales {tuple(x_scales.shape)} {x_scales.dtype} on {x_scales.device} are not f32 "
                               f"[{r.shape[0]}, {_blocks(k)}] on GPU {i}")
    s0, s1 = x_scales.stride()
    return r, x_scales.data_ptr(), s0, s1


def _out(out, shape, dtype, device, what):
    if dtype not in _IDS or dtype is E4M3:
        raise LloomHipError(2, f"{what}: {dtype} is not an output dtype (f32, f16 or bf16)")
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.dtype is not dtype or out.shape != shape or not out.is_contiguous() or out.device != device:
        raise LloomHipError(3, f"{what}: out {tuple(out.shape)} {out.dtype} on {out.device} does not fit the contiguous "
                               f"{dtype} output {tuple(shape)} on {device}")
    return out


def fp8_matmul(x, weight, weight_scales, x_scales=None, out_dtype=None, out=None):
    """x . W^T for a weight e4m3 [n, k] with f32 scales [ceil(n / 128), ceil(k / 128)]; x [.., k] f32, f16 or bf16 (brought
    into 8 bits as fp8_quantize does), or e4m3 with x_scales [rows, ceil(k / 128)].  The result [.., n] is of out_dtype (x's
    own by default, f32 for e4m3 x)."""
    i, ctx = _gpu(weight, "fp8_matmul")
    n, k = _weight(weight, weight_scales, 2, i, "fp8_matmul")
    r, xs, s0, s1 = _x(x, x_scales, i, k, "fp8_matmul")
    dtype = out_dtype or (x.dtype if x_scales is None else torch.float32 if out is None else out.dtype)
    out = _out(out, x.shape[:-1] + (n,), dtype, weight.device, "fp8_matmul")
    check(lib().lloom_hip_fp8_matmul(ctx, weight.data_ptr(), weight_scales.data_ptr(), n, k, r.data_ptr(), _IDS[r.dtype],
                                     _stride(r), xs, s0, s1, r.shape[0], out.data_ptr(), _IDS[dtype], _stream_of(i)))
    return out


def expert_plan(ids, experts):
    """The order of a step's planes by expert: ids [tokens, topk] (int32), each in [0, experts).  Planes of one expert keep
    their order.  A negative id is a plane of no expert (a padded batch); one past the last expert is too, and paged_check()
    raises.  Such planes come last, and the products' rows for them are zero."""
    i, ctx = _gpu(ids, "expert_plan")
    if ids.dtype is not torch.int32 or ids.dim() != 2:
        raise LloomHipError(2, f"expert_plan: ids {tuple(ids.shape)} {ids.dtype} are not int32 [tokens, topk]")
    ids = ids.contiguous()
    tokens, topk = ids.shape
    p = tokens * topk
    buf = ids.new_empty(2 * p + max(experts, 0) + 1)
    base = buf.data_ptr()
    check(lib().lloom_hip_expert_plan(ctx, ids.data_ptr(), tokens, topk, experts, base + 8 * p, base, base + 4 * p,
                                      _stream_of(i)))
    planes, of, starts = buf.split((p, p, experts + 1))
    return ExpertPlan(starts, planes, of)


def _index(t, i, what):
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.dim() != 1 or t.get_device() != i or not t.is_contiguous():
        raise LloomHipError(2, f"fp8_grouped_matmul: {what} {tuple(t.shape)} {t.dtype} on {t.device} is not a dense int32 "
                               f"tensor of one dimension on GPU {i}")
    return t.data_ptr()


def fp8_grouped_matmul(x, weight, weight_scales, starts, x_scales=None, gather=None, scatter=None, out_dtype=None, out=None):
    """Products grouped by expert, ragged: weights e4m3 [experts, n, k] with scales [experts, ceil(n / 128), ceil(k / 128)];
    row i with starts[e] <= i < starts[e + 1] (int32 [experts + 1], from 0, not falling) is x[gather[i]] (int32; None: x[i])
    times weight e, and is stored at out[scatter[i]] (int32, no two alike; None: out[i]).  Rows of no expert are zero.  x and
    x_scales as in fp8_matmul; the result [rows, n] has a row for each of gather, scatter or x, in that order of preference.
    With scatter, `out` may have more rows; those that scatter does not name are left as they are."""
    i, ctx = _gpu(weight, "fp8_grouped_matmul")
    n, k = _weight(weight, weight_scales, 3, i, "fp8_grouped_matmul")
    r, xs, s0, s1 = _x(x, x_scales, i, k, "fp8_grouped_matmul")
    g, c, st = _index(gather, i, "gather"), _index(scatter, i, "scatter"), _index(starts, i, "starts")
    rows = r.shape[0] if gather is None and scatter is None else (scatter if gather is None else gather).shape[0]
    if (starts.shape[0] != weight.shape[0] + 1 or (gather is None and r.shape[0] < rows)
            or (scatter is not None and scatter.shape[0] != rows)):
        raise LloomHipError(3, f"fp8_grouped_matmul: {starts.shape[0]} starts of {weight.shape[0]} experts, {rows} rows of "
                               f"{r.shape[0]}" + ("" if scatter is None else f" to {scatter.shape[0]} places"))
    dtype = out_dtype or (x.dtype if x_scales is None else torch.float32 if out is None else out.dtype)
    shape = (rows, n)
    if out is not None and scatter is not None and out.dim() == 2 and out.shape[0] > rows:
        shape = (out.shape[0], n)
    out = _out(out, shape, dtype, weight.device, "fp8_grouped_matmul")
    check(lib().lloom_hip_fp8_grouped_matmul(ctx, weight.data_ptr(), weight_scales.data_ptr(), weight.shape[0], n, k,
                                             r.data_ptr(), _IDS[r.dtype], _stride(r), xs, s0, s1, r.shape[0], st, g, c, rows,
                                             out.data_ptr(), _IDS[dtype], shape[0], _stream_of(i)))
    return out


def fp8_workspace_bytes(dtype, rows, k, x_rows=None, experts=0):
    """The workspace a product of `rows` rows takes (reserve_workspace it before a capture): x of dtype [x_rows, k], as many
    as rows by default; experts: 0 for fp8_matmul."""
    if dtype not in _IDS:
        raise LloomHipError(2, f"fp8_workspace_bytes: {dtype} is not f32, f16, bf16 or e4m3")
    out = ctypes.c_size_t()
    check(lib().lloom_hip_fp8_workspace_bytes(_IDS[dtype], rows, rows if x_rows is None else x_rows, experts, k,
                                              ctypes.byref(out)))
    return out.value
