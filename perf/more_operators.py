"""Operators of a cache that is kept short, as a user calls them, beside their plain form.

Rotary positions (rows by themselves, and fused with the write of new rows to a paged
cache), the attention weight that each cached row has been given (accumulated step by
step), and the eviction of the rows that were given least.
"""

import importlib
import math
import random

import torch

own = False

DIM = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_package = None


def _ops():
    global _package
    if _package is None:
        _package = importlib.import_module("twilight-cpu-gpu-offloading_b200")
    return _package.ops


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # One decoded token: q and k side by side in the projection's output.
        dict(name="rope_token_1", op="rope", tokens=1, heads=40, dtype="bf16", layout="half",
             dims=128, scaling="none", fused=True, far=32768),
        # The rows of a long prompt, half of each head rotated, at far positions.
        dict(name="rope_chunk_8192_part", op="rope", tokens=8192, heads=32, dtype="fp16",
             layout="interleaved", dims=64, scaling="bands", fused=False, far=1000000),
        # 16 requests decode a token each: q rotated, k rotated to its page, v to its page.
        dict(name="rope_write_16", op="rope_write", tokens=16, q_heads=32, kv_heads=8,
             dtype="bf16", layout="half", dims=128, scaling="none", page=16, pool="head",
             fused=True, records=True, far=131072),
        # A chunk with an odd rotated part, 24 query heads, the token-major pool.
        dict(name="rope_write_701_odd", op="rope_write", tokens=701, q_heads=24, kv_heads=8,
             dtype="fp16", layout="half", dims=36, scaling="linear", page=64, pool="token",
             fused=False, records=True, far=40000),
        # A large chunk of prompts out of the fused projection.
        dict(name="rope_write_8192", op="rope_write", tokens=8192, q_heads=32, kv_heads=8,
             dtype="bf16", layout="half", dims=128, scaling="yarn", page=16, pool="head",
             fused=True, records=False, far=131072),
        # One request decodes at 32k: its row's weights are added to its cache's.
        dict(name="weights_1x32k", op="weights", requests=1, chunks=0, chunk_min=0, chunk_max=0,
             ctx_min=32767, ctx_max=32767, q_heads=32, kv_heads=8, dtype="bf16", page=16,
             layout="head", window=0, last=0, lengths=1),
        # 16 requests decode, contexts from 8k to 131k.
        dict(name="weights_16_ragged", op="weights", requests=16, chunks=0, chunk_min=0,
             chunk_max=0, ctx_min=8191, ctx_max=131071, q_heads=32, kv_heads=8, dtype="bf16",
             page=16, layout="head", window=0, last=0, lengths=4),
        # Chunks and single tokens together, 24 query heads, sliding window; the last 64 rows
        # of each request are counted.
        dict(name="weights_mixed_last", op="weights", requests=16, chunks=6, chunk_min=65,
             chunk_max=701, ctx_min=0, ctx_max=4099, q_heads=24, kv_heads=8, dtype="fp16",
             page=64, layout="token", window=1000, last=64, lengths=5),
        # A whole prompt, all its rows counted.
        dict(name="weights_2048_first", op="weights", requests=1, chunks=1, chunk_min=2048,
             chunk_max=2048, ctx_min=0, ctx_max=0, q_heads=32, kv_heads=8, dtype="bf16",
             page=16, layout="head", window=0, last=0, lengths=1),
        # The last chunk of a 32k prompt.
        dict(name="weights_2048_to_32k", op="weights", requests=1, chunks=1, chunk_min=2048,
             chunk_max=2048, ctx_min=30720, ctx_max=30720, q_heads=32, kv_heads=8, dtype="bf16",
             page=16, layout="head", window=0, last=0, lengths=1),
        # One request, one layer, a few rows over its budget: what a decoding loop does often.
        dict(name="evict_1_few", op="evict", requests=1, layers=1, kv_heads=8, ctx_min=4160,
             ctx_max=4160, keep=4096, sink=4, recent=64, fresh=64, gone=5000, dtype="bf16",
             page=16, layout="head", lengths=1),
        # Prompts of up to 16k are cut to 2048 rows in four layers at once.
        dict(name="evict_4_layers_cut", op="evict", requests=4, layers=4, kv_heads=8,
             ctx_min=2000, ctx_max=16384, keep=2048, sink=64, recent=256, fresh=512, gone=0,
             dtype="bf16", page=16, layout="head", lengths=6),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("rope", "rope_write", "rope_write", "token", "chunk", "chunk", "evict",
                       "evict"))
    dtype = rng.choice(("bf16", "fp16"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    layout = rng.choice(("head", "token"))
    lengths = rng.randrange(1 << 20)
    if kind in ("rope", "rope_write"):
        case = dict(op=kind, tokens=_spread(rng, 1, 8192), dtype=dtype,
                    layout=rng.choice(("half", "interleaved")),
                    dims=rng.choice((128, 128, 64, 32, 2 * rng.randint(1, 64))),
                    scaling=rng.choice(("none", "linear", "bands", "yarn")),
                    fused=rng.random() < 0.5, far=_spread(rng, 100, 1000000))
        if kind == "rope":
            return dict(case, heads=_spread(rng, 1, 40))
        q_heads, kv_heads = rng.choice(((32, 8), (24, 8), (16, 4), (8, 8), (14, 2), (8, 1)))
        return dict(case, q_heads=q_heads, kv_heads=kv_heads, page=page, pool=layout,
                    records=rng.random() < 0.5)
    if kind == "evict":
        requests = _spread(rng, 1, 8)
        ctx = _spread(rng, 16, 65536 // requests)
        sink = rng.choice((0, 1, 4, 64))
        recent = rng.choice((0, 1, 32, 256))
        return dict(op="evict", requests=requests, layers=rng.choice((1, 1, 2, 4)),
                    kv_heads=rng.choice((1, 2, 4, 8)), ctx_min=rng.randint(0, ctx), ctx_max=ctx,
                    keep=max(sink + recent, _spread(rng, 1, ctx)), sink=sink, recent=recent,
                    fresh=rng.randint(0, ctx), gone=rng.choice((0, rng.randint(1, 20000))),
                    dtype=dtype, page=page, layout=layout, lengths=lengths)
    q_heads, kv_heads = rng.choice(((32, 8), (32, 8), (64, 8), (24, 8), (16, 4), (8, 8), (14, 2),
                                    (8, 1)))
    window = rng.choice((0, 0, 0, _spread(rng, 16, 4096)))
    if kind == "token":
        requests = _spread(rng, 1, 256)
        top = _spread(rng, 16, min(131071, (1 << 20) // requests))
        return dict(op="weights", requests=requests, chunks=0, chunk_min=0, chunk_max=0,
                    ctx_min=_spread(rng, 1, top), ctx_max=top, q_heads=q_heads,
                    kv_heads=kv_heads, dtype=dtype, page=page, layout=layout, window=window,
                    last=rng.choice((0, 1)), lengths=lengths)
    requests = _spread(rng, 1, 24)
    chunks = rng.randint(1, requests)
    chunk = _spread(rng, 2, 2048 // requests)
    ctx = _spread(rng, 1, min(30720, (1 << 26) // (requests * chunk)))
    return dict(op="weights", requests=requests, chunks=chunks, chunk_min=rng.randint(1, chunk),
                chunk_max=chunk, ctx_min=rng.randint(0, ctx), ctx_max=ctx,
                q_heads=min(q_heads, 32), kv_heads=kv_heads, dtype=dtype, page=page,
                layout=layout, window=window, last=rng.choice((0, 0, rng.randint(1, 100))),
                lengths=lengths)


def _lengths(case):
    """(tokens held before, new tokens) of each request."""
    rng = random.Random(case["lengths"])
    n, chunks = case["requests"], case.get("chunks", 0)
    new = [rng.randint(case["chunk_min"], case["chunk_max"]) for _ in range(chunks)]
    new += [1] * (n - chunks)
    rng.shuffle(new)
    return [rng.randint(case["ctx_min"], case["ctx_max"]) for _ in range(n)], new


def _pages(n, page):
    return -(-n // page)


def _counted(new, last):
    """The first of a request's new rows whose weights count."""
    return max(0, new - last) if last else 0


def work(case):
    op = case["op"]
    if op == "rope":
        row = DIM * 2
        return {"bytes": case["tokens"] * (2 * case["heads"] * row + 4),
                "flops": 3 * case["tokens"] * case["heads"] * case["dims"]}
    if op == "rope_write":
        t, q, k = case["tokens"], case["q_heads"], case["kv_heads"]
        return {"bytes": t * ((2 * q + 4 * k) * DIM * 2 + 12 + (8 * k if case["records"] else 0)),
                "flops": 3 * t * (q + k) * case["dims"]}
    if op == "evict":
        before, _ = _lengths(case)
        heads, total = case["layers"] * case["kv_heads"], 0
        for n in before:
            if n > case["keep"]:
                # rows past the budget that stay move: their share of all is what is kept
                moved = case["keep"] * (n - case["keep"]) // n
                total += heads * (8 * n + moved * (2 * 2 * DIM * 2 + 8)) + 4 * _pages(n, case["page"])
        return {"bytes": total + 24 * len(before), "flops": 0}
    pairs = keys = rows = 0
    for b, x in zip(*_lengths(case)):
        i0, w = _counted(x, case["last"]), case["window"]
        n = x - i0
        rows += n
        p = b + i0  # the first counted row's position
        if w:
            full = max(0, min(n, w - p - 1))
            pairs += full * p + full * (full + 1) // 2 + (n - full) * w
            keys += min(b + x, w + n - 1)
        else:
            pairs += n * p + n * (n + 1) // 2
            keys += b + x
    rows *= case["q_heads"]
    return {"bytes": keys * case["kv_heads"] * (DIM * 2 + 8) + keys // case["page"] * 4
            + rows * (DIM * 2 + 4), "flops": 2 * DIM * pairs * case["q_heads"]}


# ------------------------------------------------------------------ inputs --

def _frequencies(case):
    """(radians a position turns each pair, 64 bits; factor of the rotated pairs)."""
    dims, base = case["dims"], 500000.0
    inv = base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if case["scaling"] == "linear":
        return inv / 4.0, 1.0
    if case["scaling"] == "bands":  # long waves slowed by 8, short ones kept, a ramp between
        turns = 8192 * inv / (2 * math.pi)
        ramp = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv / 8.0 * (1 - ramp) + inv * ramp, 1.0
    if case["scaling"] == "yarn":  # the ramp over the pair's number, and a factor
        pair = lambda t: dims * math.log(32768 / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), dims - 1)
        ramp = ((torch.arange(dims // 2, dtype=torch.float64) - low)
                / max(high - low, 0.001)).clamp(0, 1)
        return inv / 4.0 * ramp + inv * (1 - ramp), 0.1 * math.log(4.0) + 1.0
    return inv, 1.0


def _pool(pages, layout, heads, page, make, lead=()):
    """A pool of pages as [.., pages, kv_heads, page, D]; the token-major one is a view."""
    if layout == "head":
        return make(*lead, pages, heads, page, DIM)
    return make(*lead, pages, page, heads, DIM).transpose(-3, -2)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(s, generator=g, device=dev, dtype=torch.float32).to(dt)  # noqa: E731
    if case["op"] in ("rope", "rope_write"):
        t = case["tokens"]
        frequencies, scale = _frequencies(case)
        first = torch.randint(0, case["far"], (1,), generator=g, device=dev, dtype=torch.int32)
        if t > 64:  # a chunk: one place after the other
            positions = first + torch.arange(t, device=dev, dtype=torch.int32)
        else:
            positions = torch.randint(0, case["far"], (t,), generator=g, device=dev,
                                      dtype=torch.int32)
        s = dict(case=case, positions=positions, frequencies=frequencies.to(dev), scale=scale)
        if case["op"] == "rope":
            x = normal(t, case["heads"] + (8 if case["fused"] else 0), DIM)
            return dict(s, x=x[:, :case["heads"]])
        q_heads, h, page = case["q_heads"], case["kv_heads"], case["page"]
        pages = _pages(t, page) + 3
        x = normal(t, q_heads + 2 * h, DIM)
        q, k, v = x.split((q_heads, h, h), 1)
        if not case["fused"]:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        pool = [_pool(pages, case["pool"], h, page,
                      lambda *n: torch.zeros(n, dtype=dt, device=dev)) for _ in range(2)]
        record = lambda kind: (torch.full((pages, h, page), 7, dtype=kind, device=dev)  # noqa: E731
                               if case["records"] else None)
        return dict(s, q=q, k=k, v=v, k_pages=pool[0], v_pages=pool[1],
                    slots=torch.randperm(pages * page, generator=g, device=dev)[:t],
                    weights=record(torch.float32), places=record(torch.int32),
                    error=torch.zeros(1, dtype=torch.int32, device=dev))

    before, new = _lengths(case)
    page, n, h = case["page"], case["requests"], case["kv_heads"]
    if case["op"] == "evict":
        new = [0] * n
    held = [_pages(b + x, page) for b, x in zip(before, new)]
    width, pages = max(max(held), 1), sum(held) + 5
    ids = torch.randperm(pages, generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    held_t = torch.tensor(held, device=dev)
    start = torch.cumsum(held_t, 0) - held_t
    col = torch.arange(width, device=dev)
    table = torch.where(col < held_t[:, None],
                        ids[(start[:, None] + col).clamp(max=pages - 1)], -1).contiguous()
    i32 = dict(dtype=torch.int32, device=dev)
    error = torch.zeros(1, **i32)

    if case["op"] == "evict":
        lead = (case["layers"],) if case["layers"] > 1 else ()
        k_pages = _pool(pages, case["layout"], h, page, normal, lead)
        v_pages = _pool(pages, case["layout"], h, page, normal, lead)
        # what each row was given: of very different sizes, nothing at all for some
        weights = torch.exp(2 * torch.randn(*lead, pages, h, page, generator=g, device=dev))
        weights *= torch.rand(weights.shape, generator=g, device=dev) > 0.1
        places = torch.zeros(*lead, pages, h, page, **i32)
        for b, held_b in enumerate(before):
            # `gone` of the tokens were evicted before, other ones for each head; the last
            # `fresh` rows came after that
            fresh = min(case["fresh"], held_b)
            old = held_b - fresh
            spots = torch.rand(*lead, h, old + case["gone"], generator=g, device=dev)
            spots = torch.cat((spots.argsort(-1)[..., :old].int(),
                               torch.arange(old + case["gone"], held_b + case["gone"], **i32)
                               .expand(*lead, h, fresh)), -1)
            j = torch.arange(held_b, device=dev)
            at = table[b, j // page].long()
            # [.., pages, h, page] at (at[j], head, j % page)
            heads = torch.arange(h, device=dev)[:, None]
            places[..., at, heads, j % page] = spots
        free = sum(held)
        stack = torch.full((pages,), -1, **i32)
        stack[:pages - free] = ids[free:]
        records = torch.stack((weights.view(torch.int32), places))
        return dict(case=case, k_pages=k_pages, v_pages=v_pages, records=records,
                    records_before=records.clone(), table=table, before=before,
                    lens=torch.tensor(before, **i32), lens_out=torch.zeros(n, **i32),
                    keep=torch.full((n,), case["keep"], **i32),
                    offsets=torch.full((n,), case["gone"], **i32),
                    offsets_out=torch.zeros(n, **i32), stack=stack,
                    count=torch.tensor([pages - free], **i32), count_out=torch.zeros(1, **i32),
                    max_len=max(before), error=error)

    total = sum(new)
    k_pages = _pool(pages, case["layout"], h, page, normal)
    # a few channels of K are much larger than the others, as in real models
    loud = torch.exp(torch.randn(4, generator=g, device=dev))
    k_pages[..., torch.randperm(DIM, generator=g, device=dev)[:4]] *= loud.to(dt)
    q = normal(total, case["q_heads"], DIM)
    cu = torch.zeros(n + 1, **i32)
    cu[1:] = torch.cumsum(torch.tensor(new, device=dev), 0)
    s = dict(case=case, q=q, k_pages=k_pages, table=table, cu_q=cu,
             kv_lens=torch.tensor([b + x for b, x in zip(before, new)], **i32),
             max_q=max(new), max_kv=max(b + x for b, x in zip(before, new)),
             weights=torch.exp(torch.randn(pages, h, page, generator=g, device=dev)),
             error=error)
    # the attention that came before left the log-sum-exp of its rows
    s["lse"] = torch.zeros(q.shape[:2], dtype=torch.float32, device=dev)
    for b, low, high, i, position, rows in _blocks(case, before, new):
        s["lse"][i:i + rows] = torch.logsumexp(
            _scores(s, b, low, high, i, position, rows, torch.float32), -1
        ).transpose(0, 1).flatten(1)
    return s


def _blocks(case, before, new):
    """The new rows in pieces: (request, first key, keys' end, first row, its position,
    rows)."""
    window, first = case["window"], 0
    for b, (old, x) in enumerate(zip(before, new)):
        for c in range(0, x, 1024):
            end = min(x, c + 1024)
            low = max(0, old + c - window + 1) if window else 0
            yield b, low, old + end, first + c, old + c, end - c
        first += x


def _scores(s, b, low, high, i, position, n, kind):
    """[kv_heads, rows, group, keys] of one piece, hidden ones -inf."""
    case = s["case"]
    h, page = case["kv_heads"], case["page"]
    j = torch.arange(low, high, device=s["q"].device)
    k = s["k_pages"][s["table"][b, j // page].long(), :, j % page].to(kind)  # [keys, h, D]
    q = s["q"][i:i + n].to(kind).view(n, h, -1, DIM).transpose(0, 1)
    score = (q.reshape(h, -1, DIM) @ k.permute(1, 2, 0)).view(h, n, -1, high - low)
    score /= math.sqrt(DIM)
    gap = torch.arange(position, position + n, device=j.device)[:, None] - j
    hide = (gap < 0) | (gap >= case["window"]) if case["window"] else gap < 0
    return score.masked_fill_(hide[:, None], -math.inf)


# --------------------------------------------------------------------- run --

def run(s):
    case = s["case"]
    op = case["op"]
    if op == "rope":
        if own:
            return _ops().rope(s["x"], s["positions"], s["frequencies"], layout=case["layout"],
                               scale=s["scale"])
        return _plain_rope(s["x"], s)
    if op == "rope_write":
        if own:
            q = _ops().paged_rope_write(s["q"], s["k"], s["v"], s["positions"], s["slots"],
                                        s["frequencies"], s["k_pages"], s["v_pages"],
                                        layout=case["layout"], scale=s["scale"],
                                        row_weights=s["weights"], row_positions=s["places"],
                                        error_flag=s["error"])
        else:
            q = _plain_rope_write(s)
        out = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if case["records"]:
            out.update(weights=s["weights"], places=s["places"])
        return out
    if op == "weights":
        if own:
            _ops().paged_weights(s["q"], s["k_pages"], s["table"], s["cu_q"], s["kv_lens"],
                                 s["lse"], s["weights"], max_q_len=s["max_q"],
                                 max_kv_len=s["max_kv"], window=case["window"],
                                 last=case["last"], error_flag=s["error"])
        else:
            _plain_weights(s)
        return s["weights"]
    # an eviction moves the rows' records: those of the pass before are put back first, so
    # that each pass chooses among the same rows
    s["records"].copy_(s["records_before"])
    if own:
        _ops().paged_evict(s["k_pages"], s["v_pages"], s["records"][0].view(torch.float32),
                           s["records"][1], s["table"], s["lens"], s["keep"], s["offsets"],
                           max_len=s["max_len"], sink=case["sink"], recent=case["recent"],
                           lens_out=s["lens_out"], offsets_out=s["offsets_out"],
                           free_pages=s["stack"], free_count=s["count"],
                           free_count_out=s["count_out"], error_flag=s["error"])
    else:
        _plain_evict(s)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"],
            "weights": s["records"][0].view(torch.float32), "places": s["records"][1],
            "lens": s["lens_out"], "offsets": s["offsets_out"], "stack": s["stack"],
            "count": s["count_out"]}


def _plain_rope(x, s):
    """Pair (a, b) of a row at position p: (a cos - b sin, b cos + a sin), angle p times the
    pair's frequency."""
    dims = s["case"]["dims"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos = (torch.cos(angle) * s["scale"]).float()[:, None]
    sin = (torch.sin(angle) * s["scale"]).float()[:, None]
    out = x.float()
    if s["case"]["layout"] == "half":
        a, b = out[..., :dims // 2], out[..., dims // 2:dims]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = out[..., 0:dims:2], out[..., 1:dims:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, out[..., dims:]), -1).to(x.dtype)


def _plain_rope_write(s):
    page, slots = s["case"]["page"], s["slots"]
    s["k_pages"][slots // page, :, slots % page] = _plain_rope(s["k"], s)
    s["v_pages"][slots // page, :, slots % page] = s["v"]
    if s["case"]["records"]:
        s["weights"][slots // page, :, slots % page] = 0.0
        s["places"][slots // page, :, slots % page] = s["positions"][:, None]
    return _plain_rope(s["q"], s)


def _plain_weights(s):
    case, q = s["case"], s["q"]
    h, page, t = case["kv_heads"], case["page"], q.shape[0]
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    n, mk = len(kv), s["max_kv"]
    # a bound of the counted rows of a request
    mq = min(s["max_q"], case["last"]) if case["last"] else s["max_q"]
    j = torch.arange(mk, device=q.device)
    at = s["table"][:, j // page].long().clamp(min=0)
    held = j < kv[:, None]
    k = s["k_pages"][at, :, j % page].float()  # [n, mk, h, D]
    # the last mq rows of each request
    i = torch.arange(mq, device=q.device) - mq + (cu[1:] - cu[:-1])[:, None]
    row = (cu[:-1, None] + i).clamp(0, t - 1)
    r = case["q_heads"] // h
    x = q[row].float().view(n, mq, h, r, DIM).permute(0, 2, 1, 3, 4).reshape(n, h, mq * r, DIM)
    score = torch.matmul(x, k.permute(0, 2, 3, 1)).view(n, h, mq, r, mk)
    score.mul_(1.0 / math.sqrt(DIM))
    lse = s["lse"][row].view(n, mq, h, r).permute(0, 2, 1, 3)[..., None]
    p = (kv - mq)[:, None] + torch.arange(mq, device=q.device)
    seen = (j <= p[..., None]) & (i >= 0)[..., None]
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    score.sub_(lse).exp_().masked_fill_(~seen[:, None, :, None], 0.0)
    added = score.sum((2, 3)).transpose(1, 2)  # [n, mk, h]
    s["weights"][at[held], :, (j % page).expand(n, mk)[held]] += added[held]


def _plain_evict(s):
    case = s["case"]
    page, keep, gone = case["page"], case["keep"], case["gone"]
    weights, places = s["records"][0].view(torch.float32), s["records"][1]
    lead = (case["layers"],) if case["layers"] > 1 else ()
    dev = weights.device
    heads = torch.arange(case["kv_heads"], device=dev)[:, None]
    free = s["count"].long()
    for b, n in enumerate(s["before"]):
        if n <= keep:
            continue
        j = torch.arange(n, device=dev)
        at = (s["table"][b, j // page].long(), heads, j % page)
        w, p = weights[(..., *at)], places[(..., *at)]  # [.., h, n]
        fixed = (p < case["sink"]) | (p >= n + gone - case["recent"])
        order = torch.where(fixed, math.inf, w).sort(dim=-1, descending=True, stable=True).indices
        stays = torch.zeros(*lead, case["kv_heads"], n, dtype=torch.bool, device=dev)
        stays.scatter_(-1, order[..., :keep], True)
        # the i-th row past the budget that stays goes to the i-th place left within it
        *unit, to = torch.nonzero(~stays[..., :keep], as_tuple=True)
        source = torch.nonzero(stays[..., keep:], as_tuple=True)[-1] + keep
        spot = lambda x: (*unit[:-1], s["table"][b, x // page].long(), unit[-1], x % page)  # noqa: E731
        for pool in (s["k_pages"], s["v_pages"], weights, places):
            pool[spot(to)] = pool[spot(source)]
        # pages past the last row that stays
        back = s["table"][b, _pages(keep, page):_pages(n, page)]
        s["stack"][free + torch.arange(back.numel(), device=dev)] = back
        free = free + back.numel()
    s["lens_out"].copy_(torch.minimum(s["lens"], s["keep"]))
    s["offsets_out"].copy_(s["offsets"] + s["lens"] - s["lens_out"])
    s["count_out"].copy_(free)


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    """Rotations as products of complex numbers, weights request by request, in 64 bits; an
    eviction only moves values."""
    if case["op"] == "evict":
        return None
    s = prepare(case, seed)
    if case["op"] == "weights":
        before, new = _lengths(case)
        h, page = case["kv_heads"], case["page"]
        out = s["weights"].double()
        for b, low, high, i, position, rows in _blocks(case, before, new):
            skip = max(0, before[b] + _counted(new[b], case["last"]) - position)
            if skip >= rows:
                continue
            e = _scores(s, b, low, high, i, position, rows, torch.float64)
            z = s["lse"][i:i + rows].double().view(rows, h, -1).transpose(0, 1)
            e.sub_(z[..., None]).exp_()
            e[:, :skip] = 0.0
            j = torch.arange(low, high, device=out.device)
            out[s["table"][b, j // page].long(), :, j % page] += e.sum((1, 2)).T
        return out

    turn = torch.polar(torch.full((), float(s["scale"]), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * s["frequencies"])[:, None]
    dims = case["dims"]

    def rotate(x):
        x = x.double()
        pairs = (x[..., :dims].unflatten(-1, (2, dims // 2)).transpose(-1, -2)
                 if case["layout"] == "half" else x[..., :dims].unflatten(-1, (dims // 2, 2)))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = y.transpose(-1, -2) if case["layout"] == "half" else y
        return torch.cat((y.flatten(-2), x[..., dims:]), -1)

    if case["op"] == "rope":
        return rotate(s["x"])
    page, slots = case["page"], s["slots"]
    k_pages = s["k_pages"].double()
    k_pages[slots // page, :, slots % page] = rotate(s["k"])
    out = {"q": rotate(s["q"]), "k_pages": k_pages, "v_pages": None}
    if case["records"]:
        out.update(weights=None, places=None)
    return out
