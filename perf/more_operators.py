"""What the 8-bit floating-point operators' speed is measured on: the products with e4m3 weights that have a scale for each
block of 128 x 128, dense and grouped by expert, and what stands between them, in each operator's plain form (elementary
torch operations) and, where `own` is set, as calls of lloom_amd.

Kinds of case:
  quantize  rows of activations into e4m3, a scale (a power of two) for each 128 values of a row
  gate      silu(gate) * up into the same
  matmul    y = x . W^T, x f32, f16 or bf16 (quantized within the call) or e4m3 rows with their scales
  plan      planes (token, slot) in the order of their experts, and where each expert's begin
  grouped   the planes' rows through their experts' weights, `up`: rows of x gathered by token, `down`: e4m3 rows in the
            experts' order, the results scattered to their planes

A block's scale is 2^e with the least e >= -126 for which the block's largest finite value is at most 448 * 2^e, 1 for a
block of zeros. A division by it is exact, so the nearest e4m3 number is the same in any arithmetic.
"""
import math
import random

import torch

own = False

DEV = "cuda"
ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------- the cases --

def _rows(kind, name, rows, k, act):
    return {"name": name, "kind": kind, "rows": rows, "k": k, "act": act}


def _matmul(name, m, n, k, act, out):
    return {"name": name, "kind": "matmul", "m": m, "n": n, "k": k, "act": act, "out": out}


def _plan(name, tokens, topk, experts, padded=0):
    return {"name": name, "kind": "plan", "tokens": tokens, "topk": topk, "experts": experts, "padded": padded}


def _grouped(name, way, tokens, topk, experts, n, k, act, out):
    return {"name": name, "kind": "grouped", "way": way, "tokens": tokens, "topk": topk, "experts": experts, "n": n, "k": k,
            "act": act, "out": out}


def listed():
    return [
        # one user's token, and a batch of prompts, before products that share it
        _rows("quantize", "quantize_1_f16", 1, 2048, "f16"),
        _rows("quantize", "quantize_8192_bf16", 8192, 4096, "bf16"),
        # between the two products of a layer: an odd number of rows and a last block of 96, and a batch of prompts
        _rows("gate", "gate_37_f32", 37, 1376, "f32"),
        _rows("gate", "gate_8192_f16", 8192, 4096, "f16"),
        # one user's token through the decode benchmark's weight
        _matmul("matmul_1_f16", 1, 6144, 2048, "f16", "f16"),
        # a prompt of no round length through the prefill benchmark's
        _matmul("matmul_509_f32", 509, 8192, 2048, "f32", "f32"),
        # a batch of prompts
        _matmul("matmul_8192_bf16", 8192, 8192, 8192, "bf16", "bf16"),
        # a padded decode batch, and a batch of prompts
        _plan("plan_decode_32", 32, 8, 128, padded=5),
        _plan("plan_prompt_8192", 8192, 8, 128),
        # the routed-expert benchmark's layer in decode: gate and up side by side, few rows an expert
        _grouped("up_decode_32_bf16", "up", 32, 8, 128, 1536, 2048, "bf16", "bf16"),
        # its prefill: ragged tens of rows an expert, back to the planes
        _grouped("down_prompt_512_f32", "down", 512, 8, 128, 2048, 768, "f32", "f32"),
        # a batch of prompts
        _grouped("up_prompt_8192_f16", "up", 8192, 8, 64, 2048, 2048, "f16", "f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "gate", "matmul", "matmul", "matmul", "plan", "grouped", "grouped", "grouped"])
    act = rng.choice(list(ACT))
    if kind in ("quantize", "gate"):
        rows = _log(rng, 1, 8192)
        return {"kind": kind, "rows": rows, "k": 16 * _log(rng, 1, min(512, (1 << 21) // rows)), "act": act}
    if kind == "matmul":
        m, n, k = _log(rng, 1, 8192), _log(rng, 16, 8192), 16 * _log(rng, 1, 512)
        return {"kind": kind, "m": m, "n": n, "k": k, "act": rng.choice([act, "e4m3"]), "out": rng.choice(list(ACT))}
    tokens, topk, experts = _log(rng, 1, 8192), rng.randint(1, 8), _log(rng, 4, 128)
    topk = min(topk, experts)
    if kind == "plan":
        return {"kind": kind, "tokens": tokens, "topk": topk, "experts": experts, "padded": rng.choice([0, tokens // 7])}
    n, k = 8 * _log(rng, 8, 256), 16 * _log(rng, 8, 128)
    # the plain form pads every expert's rows to the longest one's
    experts = min(experts, max(topk, 4, (1 << 28) // (n * k)))
    return {"kind": kind, "way": rng.choice(["up", "down"]), "tokens": tokens, "topk": topk, "experts": experts, "n": n, "k": k,
            "act": act, "out": rng.choice(list(ACT))}


# --------------------------------------------------------------- the inputs --

def _blocks(t):
    """t [.., k] with its last dimension in blocks of 128, the last one filled with zeros."""
    k = t.shape[-1]
    return torch.nn.functional.pad(t, (0, -k % 128)).unflatten(-1, (-1, 128))


def _scale_of(largest):
    """The power of two of a block whose largest value is `largest` (f32)."""
    bits = largest.view(torch.int32)
    e = (((bits + 0x1FFFFF) >> 23) - 8).clamp(min=1)
    return torch.where(largest > 0, (e << 23).view(torch.float32), 1.0)


def _quantized(x):
    """Rows of x into e4m3 and their scales."""
    x = x.float()
    b = _blocks(x)
    size = b.abs()
    s = _scale_of(torch.where(size < math.inf, size, 0.0).amax(-1))
    q = (b / s[..., None]).flatten(-2)[..., :x.shape[-1]]
    return q.to(E4M3), s


def _weights(gen, experts, n, k):
    """A checkpoint's weights: e4m3 with f32 scales of 128 x 128 blocks, of any value."""
    q = torch.empty(experts, n, k, dtype=E4M3, device=DEV)
    for e in range(experts):
        q[e] = torch.randn(n, k, device=DEV, generator=gen).mul_(100.0).clamp_(-448.0, 448.0).to(E4M3)
    s = torch.rand(experts, -(-n // 128), -(-k // 128), device=DEV, generator=gen).add_(0.5).mul_(0.01 / math.sqrt(k))
    return q, s


def _ids(case, gen):
    """topk different experts of each token, some experts liked more than others; padded tokens have none."""
    tokens, experts = case["tokens"], case["experts"]
    liked = torch.randn(experts, device=DEV, generator=gen).mul_(0.5)
    ids = (torch.randn(tokens, experts, device=DEV, generator=gen) + liked).topk(case["topk"], 1).indices.int()
    if case.get("padded"):
        ids[tokens - case["padded"]:] = -1
    return ids


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype):
        return torch.randn(*shape, device=DEV, generator=gen).to(dtype)

    kind = case["kind"]
    s = {"kind": kind}
    if kind == "plan":
        return {**s, "ids": _ids(case, gen), "experts": case["experts"]}
    if kind in ("quantize", "gate"):
        s["x"] = normal(case["rows"], case["k"], dtype=ACT[case["act"]])
        if kind == "gate":
            s["up"] = normal(case["rows"], case["k"], dtype=ACT[case["act"]])
        return s
    n, k, s["out"] = case["n"], case["k"], ACT[case["out"]]
    if kind == "matmul":
        w, ws = _weights(gen, 1, n, k)
        s.update(w=w[0], ws=ws[0], xs=None)
        if case["act"] == "e4m3":
            s["x"], s["xs"] = _quantized(normal(case["m"], k, dtype=torch.float32))
        else:
            s["x"] = normal(case["m"], k, dtype=ACT[case["act"]])
        return s
    w, ws = _weights(gen, case["experts"], n, k)
    plan = _plain_plan(_ids(case, gen), case["experts"])
    planes = case["tokens"] * case["topk"]
    s.update(w=w, ws=ws, starts=plan["starts"], xs=None, gather=None, scatter=None,
             most=int((plan["starts"][1:] - plan["starts"][:-1]).max()))
    if case["way"] == "up":
        s.update(x=normal(case["tokens"], k, dtype=ACT[case["act"]]), gather=plan["tokens"])
    else:
        s["x"], s["xs"] = _quantized(normal(planes, k, dtype=ACT[case["act"]]))
        s["scatter"] = plan["planes"]
    return s


# ------------------------------------------------------------ the operators --

def _plain_plan(ids, experts):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    ordered, planes = torch.sort(key, stable=True)
    starts = torch.searchsorted(ordered, torch.arange(experts + 1, device=DEV))
    return {"starts": starts.int(), "planes": planes.int(), "tokens": (planes // ids.shape[1]).int()}


def _values(q, s):
    """What e4m3 rows and their scales stand for, in f32."""
    return (_blocks(q.float()) * s[..., None]).flatten(-2)[..., :q.shape[-1]]


def _weight_values(q, s):
    """What e4m3 weights and the scales of their blocks stand for, in f32."""
    n, k = q.shape[-2:]
    s = s.repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    return q.float() * s


def _x_values(s):
    return _values(*(_quantized(s["x"]) if s["xs"] is None else (s["x"], s["xs"])))


def _plain_grouped(s):
    """Every expert's rows side by side, as many as the longest has, in one batched product."""
    x, starts = _x_values(s), s["starts"].long()
    w = _weight_values(s["w"], s["ws"])
    if s["gather"] is not None:
        x = x[s["gather"].long()]
    rows, experts = x.shape[0], w.shape[0]
    row = torch.arange(rows, device=DEV)
    who = torch.searchsorted(starts, row, right=True) - 1
    ours = who < experts
    place = torch.where(ours, row - starts[who.clamp(max=experts)], 0)
    padded = torch.zeros(experts, x.shape[1], max(1, s["most"]), device=DEV)
    padded[who[ours], :, place[ours]] = x[ours]
    y = torch.bmm(w, padded)
    out = torch.zeros(rows, w.shape[1], dtype=s["out"], device=DEV)
    at = row if s["scatter"] is None else s["scatter"].long()
    out[at[ours]] = y[who[ours], :, place[ours]].to(s["out"])
    return out


def run(s):
    kind = s["kind"]
    if own:
        import lloom_amd as L

        if kind == "quantize":
            q, scales = L.fp8_quantize(s["x"])
            return {"q": q, "scales": scales}
        if kind == "gate":
            q, scales = L.fp8_silu_mul(s["x"], s["up"])
            return {"q": q, "scales": scales}
        if kind == "matmul":
            return L.fp8_matmul(s["x"], s["w"], s["ws"], x_scales=s["xs"], out_dtype=s["out"])
        if kind == "plan":
            p = L.expert_plan(s["ids"], s["experts"])
            return {"starts": p.starts, "planes": p.planes, "tokens": p.tokens}
        return L.fp8_grouped_matmul(s["x"], s["w"], s["ws"], s["starts"], x_scales=s["xs"], gather=s["gather"],
                                    scatter=s["scatter"], out_dtype=s["out"])
    if kind in ("quantize", "gate"):
        x = s["x"].float()
        if kind == "gate":
            x = x / (1.0 + torch.exp(-x)) * s["up"].float()
        q, scales = _quantized(x)
        return {"q": q, "scales": scales}
    if kind == "matmul":
        return torch.mm(_x_values(s), _weight_values(s["w"], s["ws"]).t()).to(s["out"])
    if kind == "plan":
        return _plain_plan(s["ids"], s["experts"])
    return _plain_grouped(s)


def work(case):
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
    if kind in ("quantize", "gate"):
        rows, k, blocks = case["rows"], case["k"], -(-case["k"] // 128)
        read = size[case["act"]] * rows * k * (2 if kind == "gate" else 1)
        return {"bytes": read + rows * (k + 4 * blocks), "flops": 0}
    if kind == "plan":
        planes = case["tokens"] * case["topk"]
        return {"bytes": 12 * planes + 4 * (case["experts"] + 1), "flops": 0}
    n, k = case["n"], case["k"]
    row, weight = k + 4 * (-(-k // 128)), n * k + 4 * (-(-n // 128)) * (-(-k // 128))
    if kind == "matmul":
        m = case["m"]
        x = row if case["act"] == "e4m3" else size[case["act"]] * k
        return {"bytes": m * x + weight + m * n * size[case["out"]], "flops": 2 * m * n * k}
    tokens, planes, experts = case["tokens"], case["tokens"] * case["topk"], case["experts"]
    # experts that some token takes: as if tokens liked all alike
    active = experts * (1.0 - (1.0 - case["topk"] / experts) ** tokens)
    x = planes * row if case["way"] == "down" else tokens * size[case["act"]] * k
    return {"bytes": int(x + active * weight + 4 * planes + planes * n * size[case["out"]]), "flops": 2 * planes * n * k}


def _nearest(v):
    """The e4m3 number next to each v (f64, at most 448 in size), by arithmetic: steps of 2^-3 of its power of two, 2^-9 at
    least."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return torch.round(v / step) * step


def _exact_rows(x):
    """e4m3 values and scales of rows of x (f64) from the definition."""
    rows, k = x.shape
    q, scales = torch.empty_like(x), torch.empty(rows, -(-k // 128), dtype=torch.float64, device=DEV)
    for b in range(scales.shape[1]):
        part = x[:, 128 * b:128 * b + 128]
        top, e = torch.frexp(part.abs().amax(1) / 448.0)  # top in [1/2, 1): 2^e is enough, 2^(e - 1) for 1/2 itself
        e = torch.where(top == 0.5, e - 1, e).clamp(min=-126)
        s = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), 1.0)
        scales[:, b] = s
        q[:, 128 * b:128 * b + 128] = _nearest(part / s[:, None])
    return q, scales


def _exact_x(s):
    if s["xs"] is None:
        q, scales = _exact_rows(s["x"].double())
    else:
        q, scales = s["x"].double(), s["xs"].double()
    for b in range(scales.shape[1]):
        q[:, 128 * b:128 * b + 128] *= scales[:, b:b + 1]
    return q


def _exact_weight(q, scales):
    w = q.double()
    for i in range(scales.shape[0]):
        for b in range(scales.shape[1]):
            w[128 * i:128 * i + 128, 128 * b:128 * b + 128] *= scales[i, b].double()
    return w


def exact(case, seed):
    """The definitions in 64 bits, one block and one expert after another."""
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return None
    if case["kind"] in ("quantize", "gate"):
        x = s["x"].double()
        if case["kind"] == "gate":
            x = x * torch.sigmoid(x) * s["up"].double()
        q, scales = _exact_rows(x)
        return {"q": q, "scales": scales}
    x = _exact_x(s)
    if case["kind"] == "matmul":
        return x @ _exact_weight(s["w"], s["ws"]).t()
    starts = s["starts"].tolist()
    rows = case["tokens"] * case["topk"]
    y = torch.zeros(rows, case["n"], dtype=torch.float64, device=DEV)
    for e in range(case["experts"]):
        i = torch.arange(starts[e], starts[e + 1], device=DEV)
        if not len(i):
            continue
        source = i if s["gather"] is None else s["gather"][i].long()
        y[i if s["scatter"] is None else s["scatter"][i].long()] = x[source] @ _exact_weight(s["w"][e], s["ws"][e]).t()
    return y
