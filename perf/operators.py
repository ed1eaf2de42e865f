"""What the paged-cache operators' speed is measured on: the calls a program that serves a packed model makes around its
projections, in each operator's plain form (elementary torch operations) and, where `own` is set, as calls of lloom_amd.

Kinds of case:
  plan    the block tables, slots and positions of one step's new tokens, from the requests' lengths
  append  one layer's new k and v rows into the pages of the cache
  attend  one layer's attention of the new tokens over the pages: one token a request (decode), chunks of prompts, or
          both, over everything before or over a sliding window and the first few tokens

A cache is k [pages, kv_heads, page, head_dim] and v [pages, kv_heads, head_dim, page], both f16. A request's lengths are
drawn from the case alone; what the tensors hold, and which pages a request owns, from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
ACT = {"f32": torch.float32, "f16": torch.float16}


# ---------------------------------------------------------------- the cases --

def _plan(name, requests, cached, page, chunks=0, chunk=1, lens=1):
    return {"name": name, "kind": "plan", "requests": requests, "cached": cached, "page": page, "chunks": chunks,
            "chunk": chunk, "lens": lens}


def _append(name, requests, cached, page, kv_heads, dim, act, chunks=0, chunk=1, lens=1):
    return {"name": name, "kind": "append", "requests": requests, "cached": cached, "page": page, "chunks": chunks,
            "chunk": chunk, "lens": lens, "kv_heads": kv_heads, "dim": dim, "act": act}


def _attend(name, requests, cached, page, kv_heads, group, dim, act, chunks=0, chunk=1, window=0, sinks=0, lens=1):
    return {"name": name, "kind": "attend", "requests": requests, "cached": cached, "page": page, "chunks": chunks,
            "chunk": chunk, "lens": lens, "kv_heads": kv_heads, "group": group, "dim": dim, "act": act,
            "window": window, "sinks": sinks}


def listed():
    # 16 query and 4 key heads of 128 are the projections of the decoder-layer benchmark (q 2048, k and v 512)
    return [
        # a decode step of 64 requests, and a step that mixes 200 decoding requests with 24 prompts' chunks
        _plan("plan_decode_64", 64, 8191, 16),
        _plan("plan_mixed_224", 224, 8191, 16, chunks=24, chunk=509),
        # the same two kinds of step, as the cache sees them
        _append("append_decode_64_f32", 64, 8191, 16, 4, 128, "f32"),
        _append("append_prompt_8192_f16", 4, 0, 64, 8, 128, "f16", chunks=4, chunk=2048),
        # one user at the start of a conversation: latency
        _attend("decode_1_f32", 1, 640, 16, 4, 4, 128, "f32"),
        # a full decode batch, conversations of all lengths
        _attend("decode_32_f16", 32, 8191, 16, 4, 4, 128, "f16"),
        # one user deep in a long document
        _attend("decode_long_f16", 1, 131071, 64, 8, 4, 128, "f16", lens=0),
        # a model whose layers see the last 1024 tokens and four first ones, heads of 64
        _attend("decode_window_64_f32", 64, 32767, 32, 8, 4, 64, "f32", window=1024, sinks=4),
        # a whole prompt at once
        _attend("prompt_4096_f16", 1, 0, 64, 4, 4, 128, "f16", chunks=1, chunk=4096),
        # pieces of four prompts whose earlier pieces are in the cache
        _attend("chunk_509_f32", 4, 8000, 32, 4, 4, 128, "f32", chunks=4, chunk=509),
        # the same with a window
        _attend("chunk_window_f16", 2, 8192, 16, 4, 4, 128, "f16", chunks=2, chunk=2048, window=1024, sinks=4),
        # a step of continuous batching: fourteen requests decode while two prompts are read
        _attend("mixed_16_f16", 16, 4000, 16, 4, 4, 128, "f16", chunks=2, chunk=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend"])
    page, lens = rng.choice([16, 32, 64, 128]), rng.randrange(1, 1 << 20)
    if kind == "plan":
        requests = _log(rng, 1, 224)
        return {"kind": kind, "requests": requests, "cached": _log(rng, 1, 8191), "page": page,
                "chunks": rng.randint(0, min(requests, 24)), "chunk": _log(rng, 2, 509), "lens": lens}
    kv_heads, dim, act = rng.randint(1, 8), rng.choice([64, 96, 128, 256]), rng.choice(["f16", "f32"])
    if kind == "append":
        requests = _log(rng, 1, 64)
        chunks = rng.randint(0, min(requests, 4))
        dim = min(dim, 128)
        return {"kind": kind, "requests": requests, "cached": _log(rng, 1, 8191), "page": page, "chunks": chunks,
                "chunk": _log(rng, 2, 2048), "lens": lens, "kv_heads": kv_heads, "dim": dim, "act": act}
    requests, cached, group = _log(rng, 1, 64), _log(rng, 1, 32767), rng.randint(1, 8)
    chunks = rng.choice([0, 0, requests, rng.randint(0, min(requests, 4))])
    chunk = _log(rng, 2, 2048)
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    sinks = rng.randint(0, 8) if window else 0
    # within what the listed cases cost: the pages of all requests, and the pairs of the chunks' tokens
    requests = max(1, min(requests, (1 << 27) // ((cached + chunk) * kv_heads * dim)))
    chunks = min(chunks, requests)
    while chunks and requests * chunk * (cached + chunk) * kv_heads * group * dim > 1 << 34:
        if chunk > 8:
            chunk //= 2
        else:
            cached = max(1, cached // 2)
    return {"kind": kind, "requests": requests, "cached": cached, "page": page, "chunks": chunks, "chunk": chunk,
            "lens": lens, "kv_heads": kv_heads, "group": group, "dim": dim, "act": act, "window": window,
            "sinks": sinks}


def _lengths(case):
    """Cached and new tokens of each request: cached lengths spread over their logarithm up to the case's, the chunks at
    places of their own among the decoding requests, each a little shorter than the one before."""
    rng, n = random.Random(case["lens"]), case["requests"]
    most = case["cached"]
    cached = [most if case["lens"] == 0 or b == 0 else int(math.exp(rng.uniform(0, math.log(most + 1)))) if most else 0
              for b in range(n)]
    new = [1] * n
    for i, b in enumerate(sorted(rng.sample(range(n), case["chunks"]))):
        new[b] = max(1, case["chunk"] - 3 * i) if case["cached"] else case["chunk"]
    return cached, new


def _pages(n, page):
    return -(-n // page)


# --------------------------------------------------------------- the inputs --

def _tables(cached, new, page, gen, spare):
    """The pages of every request as a server's pool hands them out: any page, in any order."""
    need = [_pages(c, page) for c in cached]
    take = [_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new)]
    most = max(a + b for a, b in zip(need, take))
    pages = sum(need) + sum(take) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    tables = torch.zeros(len(cached), most, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, order[at:], take, pages


def _grown(tables, free, cached, take, page):
    """The tables once the new tokens' pages are in them."""
    tables, at = tables.clone(), 0
    for b, t in enumerate(take):
        tables[b, _pages(cached[b], page):_pages(cached[b], page) + t] = free[at:at + t]
        at += t
    return tables


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = _lengths(case)
    page, tokens = case["page"], sum(new)
    tables, free, take, pages = _tables(cached, new, page, host, spare=7)
    s = {"kind": case["kind"], "page": page, "tokens": tokens}
    ints = lambda v: torch.tensor(v, dtype=torch.int32).to(DEV)  # noqa: E731
    if case["kind"] == "plan":
        s.update(cached=ints(cached), new=ints(new), tables=tables.to(DEV), free=free.to(DEV))
        return s
    h, d, act = case["kv_heads"], case["dim"], ACT[case["act"]]
    grown = _grown(tables, free, cached, take, page)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    def normal(*shape, dtype=act, std=1.0):
        return torch.randn(*shape, device=DEV, generator=gen).mul_(std).to(dtype)

    s.update(k_cache=normal(pages, h, page, d, dtype=torch.float16), v_cache=normal(pages, h, d, page, dtype=torch.float16))
    if case["kind"] == "append":
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)])
        who = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
        s.update(k=normal(tokens, h, d), v=normal(tokens, h, d),
                 slots=(grown[who, pos // page].long() * page + pos % page).to(DEV))
        return s
    # queries that find some keys: scores of a standard deviation of two
    s.update(q=normal(tokens, h * case["group"], d, std=2.0), tables=grown.to(DEV), starts=ints(starts),
             lens=ints([c + n for c, n in zip(cached, new)]), window=case["window"], sinks=case["sinks"],
             longest=max(new))
    return s


# ------------------------------------------------------------ the operators --

def _plain_plan(s):
    cached, new, tables, free, page, tokens = s["cached"].long(), s["new"].long(), s["tables"], s["free"], s["page"], s["tokens"]
    starts = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    lens = cached + new
    held = (cached + page - 1) // page
    take = (lens + page - 1) // page - held
    off = torch.cumsum(take, 0) - take
    column = torch.arange(tables.shape[1], device=DEV)
    fresh = (column >= held[:, None]) & (column < (held + take)[:, None])
    got = free[(off[:, None] + column - held[:, None]).clamp(0, free.numel() - 1)]
    tables.copy_(torch.where(fresh, got, tables))
    token = torch.arange(tokens, device=DEV)
    who = torch.searchsorted(starts, token, right=True) - 1
    pos = cached[who] + token - starts[who]
    slots = tables[who, pos // page].long() * page + pos % page
    return {"tables": tables, "starts": starts.int(), "lens": lens.int(), "positions": pos.int(), "slots": slots,
            "taken": take.sum().int().reshape(1)}


def _plain_append(s):
    page, slots = s["page"], s["slots"]
    at, off = slots // page, slots % page
    s["k_cache"][at, :, off] = s["k"].half()
    s["v_cache"][at, :, :, off] = s["v"].half()
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s, wide):
    """The definition over padded requests, in the type `wide`: every request's keys side by side, and as many rows as
    the longest chunk has."""
    q, tables, starts, lens = s["q"], s["tables"].long(), s["starts"].long(), s["lens"].long()
    requests, (pages, h, page, d) = tables.shape[0], s["k_cache"].shape
    k = s["k_cache"][tables].to(wide).permute(0, 2, 1, 3, 4).reshape(requests, h, -1, d)
    v = s["v_cache"][tables].to(wide).permute(0, 2, 1, 4, 3).reshape(requests, h, -1, d)
    new, rows, group = starts[1:] - starts[:-1], s["longest"], q.shape[1] // h
    row = torch.arange(rows, device=DEV)
    padded = q[(starts[:-1, None] + row).clamp(max=q.shape[0] - 1)].to(wide)
    padded = padded.reshape(requests, rows, h, group, d).permute(0, 2, 1, 3, 4).reshape(requests, h, rows * group, d)
    scores = torch.matmul(padded, k.transpose(-1, -2).contiguous()).reshape(requests, h, rows, group, -1)
    scores *= 1.0 / math.sqrt(d)
    key, pos = torch.arange(k.shape[2], device=DEV), (lens - new)[:, None] + row
    seen = key <= pos[:, :, None]
    if s["window"]:
        seen &= (key > pos[:, :, None] - s["window"]) | (key < s["sinks"])
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_().reshape(requests, h, rows * group, -1)
    out = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(requests, h, rows, group, d)
    token = torch.arange(q.shape[0], device=DEV)
    who = torch.searchsorted(starts, token, right=True) - 1
    return out[who, :, token - starts[who]].reshape(q.shape)


def run(s):
    if own:
        import lloom_amd as L

        if s["kind"] == "plan":
            p = L.paged_plan(s["cached"], s["new"], s["tokens"], s["tables"], s["free"], s["page"])
            return {"tables": p.block_tables, "starts": p.q_start, "lens": p.seq_lens, "positions": p.positions,
                    "slots": p.slots, "taken": p.taken}
        if s["kind"] == "append":
            L.paged_append(s["k_cache"], s["v_cache"], s["k"], s["v"], s["slots"])
            return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return L.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["starts"], s["lens"],
                                 window=s["window"], sinks=s["sinks"], max_new=s["longest"])
    if s["kind"] == "plan":
        return _plain_plan(s)
    if s["kind"] == "append":
        return _plain_append(s)
    return _attention(s, torch.float32).to(s["q"].dtype)


def _seen(case):
    """Keys that any new token of a request sees, and pairs of a new token and a key that it sees, over all requests."""
    keys = pairs = 0
    cached, new = _lengths(case)
    w, k = case["window"], case["sinks"]
    for c, n in zip(cached, new):
        end = c + n
        lo = max(0, c - w + 1) if w else 0
        keys += end - lo + min(k, lo)
        for p in range(c, end):
            first = max(0, p - w + 1) if w else 0
            pairs += p + 1 - first + min(k, first)
    return keys, pairs


def work(case):
    cached, new = _lengths(case)
    tokens, requests, page = sum(new), len(new), case["page"]
    take = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
    if case["kind"] == "plan":
        return {"bytes": 16 * requests + 8 * take + 12 * tokens, "flops": 0}
    size = 4 if case["act"] == "f32" else 2
    if case["kind"] == "append":
        return {"bytes": tokens * (8 + 2 * case["kv_heads"] * case["dim"] * (size + 2)), "flops": 0}
    heads, d = case["kv_heads"] * case["group"], case["dim"]
    keys, pairs = _seen(case)
    return {"bytes": 2 * 2 * keys * case["kv_heads"] * d + 2 * tokens * heads * d * size, "flops": 4 * d * heads * pairs}


def exact(case, seed):
    """Attention in 64 bits, one request and one key head after another over the keys each token sees; the other two
    operators compute no numbers (a plan's are whole, an append's are copies rounded once)."""
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return None
    if case["kind"] == "append":
        pages, h, page, d = s["k_cache"].shape
        k = s["k_cache"].double().transpose(1, 2).reshape(pages * page, h, d)
        v = s["v_cache"].double().permute(0, 3, 1, 2).reshape(pages * page, h, d)
        k[s["slots"]], v[s["slots"]] = s["k"].double(), s["v"].double()
        return {"k_cache": k.reshape(pages, page, h, d).transpose(1, 2).contiguous(),
                "v_cache": v.reshape(pages, page, h, d).permute(0, 2, 3, 1).contiguous()}
    cached, new = _lengths(case)
    h, group, d, page = case["kv_heads"], case["group"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    tables, first = s["tables"].long(), 0
    for b, (c, n) in enumerate(zip(cached, new)):
        key = torch.arange(c + n, device=DEV)
        home, place = tables[b][key // page], key % page
        pos = torch.arange(c, c + n, device=DEV)[:, None]
        hidden = key > pos
        if case["window"]:
            hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
        for j in range(h):
            k, v = s["k_cache"][home, j, place].double(), s["v_cache"][home, j, :, place].double()
            for g in range(j * group, (j + 1) * group):
                z = torch.mm(s["q"][first:first + n, g].double(), k.t().contiguous()) / math.sqrt(d)
                w = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
                out[first:first + n, g] = torch.mm(w, v)
        first += n
    return out
