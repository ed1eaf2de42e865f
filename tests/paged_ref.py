"""The paged-cache operators from their definitions, in 64 bits on the CPU."""
import math

import torch


def pages_for(n, page):
    return -(-n // page)


def plan(cached, new, tokens, tables, free, page):
    """(q_start, seq_lens, positions, slots, taken, tables) as lists; tables is a list of lists."""
    tables = [list(t) for t in tables]
    starts, lens, pos, slots, taken = [0], [], [], [], 0
    for b, (c, n) in enumerate(zip(cached, new)):
        for t in range(c, c + n):
            blk = t // page
            if blk >= pages_for(c, page) and t % page == 0 and blk < len(tables[b]):
                at = taken + blk - pages_for(c, page)
                tables[b][blk] = free[at] if at < len(free) else -1
            pg = tables[b][blk] if blk < len(tables[b]) else -1
            pos.append(t)
            slots.append(pg * page + t % page if pg >= 0 else -1)
        taken += pages_for(c + n, page) - pages_for(c, page)
        starts.append(starts[-1] + n)
        lens.append(c + n)
    pos += [0] * (tokens - len(pos))
    slots += [-1] * (tokens - len(slots))
    return starts, lens, pos[:tokens], slots[:tokens], taken, tables


def attention(q, k_cache, v_cache, tables, q_start, seq_lens, scale, window, sinks):
    """out [tokens, heads, dim] in f64, and for a bound on a kernel's error, per output value: `mass`, the weighted mean
    of |v|, and per (token, head): `reach`, the largest scale * sum |q| |k| over the keys seen, and their number."""
    q, k_cache, v_cache = q.double().cpu(), k_cache.cpu(), v_cache.cpu()
    n, heads, dim = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    group = heads // kv_heads
    out, mass = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dim, dtype=torch.float64)
    reach, count = torch.zeros(n, heads, dtype=torch.float64), torch.zeros(n, heads)
    for b, length in enumerate(seq_lens):
        first, end = q_start[b], q_start[b + 1]
        key = torch.arange(max(length, 0))
        blk = key // page
        inside = blk < len(tables[b])
        pg = torch.tensor(tables[b])[blk.clamp(max=len(tables[b]) - 1)]
        inside &= (pg >= 0) & (pg < pages)
        key, pg = key[inside], pg[inside].long()
        for i in range(first, end):
            p = length - (end - first) + i - first
            seen = (key <= p) & ((key > p - window) | (key < sinks) if window else torch.ones_like(key, dtype=torch.bool))
            if not seen.any():
                continue
            ks, vs = k_cache[pg[seen], :, key[seen] % page].double(), v_cache[pg[seen], :, :, key[seen] % page].double()
            for h in range(heads):
                kh, vh = ks[:, h // group], vs[:, h // group]
                w = torch.softmax(scale * (kh @ q[i, h]), 0)
                out[i, h], mass[i, h] = w @ vh, w @ vh.abs()
                reach[i, h], count[i, h] = abs(scale) * (kh.abs() @ q[i, h].abs()).max(), len(ks)
    return out, mass, reach, count


def dense(s, request):
    """`attention` of one request that sees everything before it, on the tensors' device (for lengths that take too long a
    token at a time)."""
    first, end, length = s["q_start"][request], s["q_start"][request + 1], s["seq_lens"][request]
    key = torch.arange(length, device=s["q"].device)
    pages, kv_heads, page, dim = s["k"].shape
    home = s["t_tables"][request].long()[key // page]
    pos = torch.arange(length - (end - first), length, device=key.device)
    q = s["q"][first:end].double()
    heads = q.shape[1]
    out, mass = torch.empty_like(q), torch.empty_like(q)
    reach, count = torch.empty(end - first, heads), (pos + 1).float().cpu()[:, None].expand(-1, heads)
    for h in range(heads):
        j = h // (heads // kv_heads)
        k, v = s["k"][home, j, key % page].double(), s["v"][home, j, :, key % page].double()
        z = s["scale"] * torch.mm(q[:, h], k.t().contiguous())
        w = torch.softmax(z.masked_fill(key > pos[:, None], -math.inf), 1)
        out[:, h], mass[:, h] = torch.mm(w, v), torch.mm(w, v.abs())
        reach[:, h] = s["scale"] * torch.mm(q[:, h].abs(), k.abs().t().contiguous()).amax(1).cpu()
    return out.cpu(), mass.cpu(), reach, count


def bound(out, mass, reach, count, act, dim):
    """How far a kernel may be from `out`: a score is off by its sum's roundings (dim + 2 of half an f32 step of
    sum |q| |k|), by a few more where it is scaled and has the maximum taken off, and with f32 q by what two halves leave
    of q (2^-22 of a row's largest: within 2^-21 of reach for rows whose values are of like size); a weight by e^score
    (twice: it and the sum it is divided by), by its own rounding (f16: half a step; f32: two halves, 2^-22) and by
    exp2's; the sums by a rounding a key; the result by its type's."""
    f32 = torch.finfo(torch.float32).eps / 2
    score = reach * ((dim + 8) * f32 + (2.0 ** -21 if act == torch.float32 else 0.0))
    weight = torch.finfo(torch.float16).eps / 2 if act == torch.float16 else 2.0 ** -22
    rel = 2 * score + 2 * weight + (2 * count + 64) * f32
    return rel[..., None] * mass + torch.finfo(act).eps / 2 * out.abs() + 2.0 ** -24


def case(cached, new, page, kv_heads, group, dim, act, seed=0, spare=3, pad=0, device="cpu"):
    """Caches, tables and rows of requests of these lengths; what no token sees is NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [pages_for(c + n, page) for c, n in zip(cached, new)]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    blocks = max(need + [1])
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n] + [pages + 5] * (blocks - n))
        at += n
    k = torch.full((pages, kv_heads, page, dim), math.nan, dtype=torch.float16)
    v = torch.full((pages, kv_heads, dim, page), math.nan, dtype=torch.float16)
    for b, (c, n) in enumerate(zip(cached, new)):
        for i in range(pages_for(c + n, page)):
            m = min(page, c + n - i * page)
            k[tables[b][i], :, :m] = torch.randn(kv_heads, m, dim, generator=g).half()
            v[tables[b][i], :, :, :m] = torch.randn(kv_heads, dim, m, generator=g).half()
    tokens = sum(new) + pad
    q = (2 * torch.randn(tokens, kv_heads * group, dim, generator=g)).to(act)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    lens = [c + n for c, n in zip(cached, new)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return {"q": q.to(device), "k": k.to(device), "v": v.to(device), "tables": tables, "q_start": starts, "seq_lens": lens,
            "t_tables": ints(tables), "t_start": ints(starts), "t_lens": ints(lens), "scale": 1 / math.sqrt(dim)}
