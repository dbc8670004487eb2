"""The paged KV cache's operators as a user calls them, beside their plain form.

Three operators: the step plan (block tables and slot maps from request
lengths), the write of new K / V rows to their slots, and the attention of a
batch's new tokens (one each, or chunks of prompts) over the paged cache.
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
        # One decode step of 16 long requests: the smallest call there is.
        dict(name="step_decode_16", op="step", requests=16, chunks=0, chunk_max=0, finished=0,
             ctx_min=8192, ctx_max=131072, page=16, lengths=1),
        # A serving step with everything in it: prompts in chunks, decodes, requests that end.
        dict(name="step_mixed_256", op="step", requests=256, chunks=32, chunk_max=777, finished=16,
             ctx_min=1, ctx_max=8192, page=16, lengths=2),
        # The new rows of 64 decoding requests, 8 KV heads.
        dict(name="write_decode_64", op="write", tokens=64, kv_heads=8, dtype="bf16", page=16,
             layout="head", fused=False),
        # A chunk of prompts, K and V still inside the projection's output.
        dict(name="write_chunk_8192", op="write", tokens=8192, kv_heads=8, dtype="fp16", page=64,
             layout="token", fused=True),
        # One request decoding at 32k.
        dict(name="token_1x32k", op="attend", requests=1, chunks=0, chunk_min=0, chunk_max=0,
             ctx_min=32767, ctx_max=32767, q_heads=32, kv_heads=8, dtype="bf16", page=16,
             layout="head", window=0, lengths=1),
        # 16 requests decoding, contexts from 8k to 131k.
        dict(name="token_16_ragged", op="attend", requests=16, chunks=0, chunk_min=0, chunk_max=0,
             ctx_min=8191, ctx_max=131071, q_heads=32, kv_heads=8, dtype="bf16", page=16,
             layout="head", window=0, lengths=4),
        # Many short conversations, 64 query heads, the token-major pool.
        dict(name="token_256_short", op="attend", requests=256, chunks=0, chunk_min=0, chunk_max=0,
             ctx_min=1, ctx_max=2047, q_heads=64, kv_heads=8, dtype="fp16", page=16,
             layout="token", window=0, lengths=3),
        # A short follow-up question: latency counts.
        dict(name="chunk_33_over_100", op="attend", requests=1, chunks=1, chunk_min=33,
             chunk_max=33, ctx_min=100, ctx_max=100, q_heads=32, kv_heads=8, dtype="bf16",
             page=16, layout="head", window=0, lengths=1),
        # A whole prompt at once.
        dict(name="chunk_2048_first", op="attend", requests=1, chunks=1, chunk_min=2048,
             chunk_max=2048, ctx_min=0, ctx_max=0, q_heads=32, kv_heads=8, dtype="bf16",
             page=16, layout="head", window=0, lengths=1),
        # Chunks and single tokens of 16 requests in one call, 24 query heads, sliding window.
        dict(name="chunk_mixed_window", op="attend", requests=16, chunks=6, chunk_min=65,
             chunk_max=701, ctx_min=0, ctx_max=4099, q_heads=24, kv_heads=8, dtype="fp16",
             page=64, layout="token", window=1000, lengths=5),
        # The last chunk of a 32k prompt.
        dict(name="chunk_2048_to_32k", op="attend", requests=1, chunks=1, chunk_min=2048,
             chunk_max=2048, ctx_min=30720, ctx_max=30720, q_heads=32, kv_heads=8, dtype="bf16",
             page=16, layout="head", window=0, lengths=1),
        # The same with 64 query heads and larger chunks.
        dict(name="chunk_4096_to_32k", op="attend", requests=1, chunks=1, chunk_min=4096,
             chunk_max=4096, ctx_min=28672, ctx_max=28672, q_heads=64, kv_heads=8, dtype="bf16",
             page=64, layout="head", window=0, lengths=1),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("step", "write", "token", "chunk", "chunk"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    dtype = rng.choice(("bf16", "fp16"))
    layout = rng.choice(("head", "token"))
    lengths = rng.randrange(1 << 20)
    if kind == "step":
        requests = _spread(rng, 1, 512)
        chunks = rng.randint(0, requests // 2)
        return dict(op="step", requests=requests, chunks=chunks, chunk_max=_spread(rng, 2, 1024),
                    finished=rng.randint(0, (requests - chunks) // 4), ctx_min=1,
                    ctx_max=_spread(rng, 64, 65536), page=page, lengths=lengths)
    if kind == "write":
        return dict(op="write", tokens=_spread(rng, 1, 16384), kv_heads=rng.choice((1, 2, 4, 8)),
                    dtype=dtype, page=page, layout=layout, fused=rng.random() < 0.5)
    q_heads, kv_heads = rng.choice(((32, 8), (32, 8), (64, 8), (24, 8), (16, 4), (8, 8), (14, 2),
                                    (8, 1)))
    window = rng.choice((0, 0, 0, _spread(rng, 16, 4096)))
    if kind == "token":
        requests = _spread(rng, 1, 256)
        top = _spread(rng, 16, min(131071, (1 << 21) // requests))
        return dict(op="attend", requests=requests, chunks=0, chunk_min=0, chunk_max=0,
                    ctx_min=_spread(rng, 1, top), ctx_max=top, q_heads=q_heads,
                    kv_heads=kv_heads, dtype=dtype, page=page, layout=layout, window=window,
                    lengths=lengths)
    requests = _spread(rng, 1, 24)
    chunks = rng.randint(1, requests)
    chunk = _spread(rng, 2, 4096 // requests)
    ctx = _spread(rng, 1, min(32768, (1 << 27) // (requests * chunk)))
    return dict(op="attend", requests=requests, chunks=chunks, chunk_min=rng.randint(1, chunk),
                chunk_max=chunk, ctx_min=rng.randint(0, ctx), ctx_max=ctx, q_heads=q_heads,
                kv_heads=kv_heads, dtype=dtype, page=page, layout=layout, window=window,
                lengths=lengths)


def _lengths(case):
    """(tokens held before, new tokens) of each request; -1 new tokens: it has ended."""
    rng = random.Random(case["lengths"])
    n, chunks, finished = case["requests"], case["chunks"], case.get("finished", 0)
    low = case.get("chunk_min", 2)
    new = [rng.randint(low, case["chunk_max"]) for _ in range(chunks)]
    new += [-1] * finished + [1] * (n - chunks - finished)
    rng.shuffle(new)
    return [rng.randint(case["ctx_min"], case["ctx_max"]) for _ in range(n)], new


def _pages(n, page):
    return -(-n // page)


def _visible(before, new, window):
    """(query, key) pairs that the mask leaves, and the keys that any query sees."""
    if not window:
        return new * before + new * (new + 1) // 2, before + new
    full = max(0, min(new, window - before - 1))  # queries that see all before them
    pairs = full * before + full * (full + 1) // 2 + (new - full) * window
    return pairs, min(before + new, window + new - 1)


def work(case):
    if case["op"] == "write":
        row = case["kv_heads"] * DIM * 2
        return {"bytes": 4 * case["tokens"] * row + 8 * case["tokens"], "flops": 0}
    before, new = _lengths(case)
    page = case["page"]
    if case["op"] == "step":
        total = sum(max(0, x) for x in new)
        taken = sum(_pages(b + x, page) - _pages(b, page) for b, x in zip(before, new) if x > 0)
        back = sum(_pages(b, page) for b, x in zip(before, new) if x < 0)
        return {"bytes": 8 * len(new) + 8 * (taken + back) + 12 * total + 8 * len(new) + 16,
                "flops": 0}
    pairs = keys = 0
    for b, x in zip(before, new):
        p, k = _visible(b, x, case["window"])
        pairs += p
        keys += k
    rows = sum(new) * case["q_heads"]
    return {"bytes": keys * case["kv_heads"] * DIM * 4 + keys // page * 4 + rows * (DIM * 4 + 4),
            "flops": 4 * DIM * pairs * case["q_heads"]}


# ------------------------------------------------------------------ inputs --

def _pool(pages, case, make):
    """A pool of pages as [pages, kv_heads, page, D]; the token-major one is a view."""
    if case["layout"] == "head":
        return make(pages, case["kv_heads"], case["page"], DIM)
    return make(pages, case["page"], case["kv_heads"], DIM).transpose(1, 2)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(int(seed))
    if case["op"] == "write":
        t, h, page = case["tokens"], case["kv_heads"], case["page"]
        dt = DTYPES[case["dtype"]]
        pages = _pages(t, page) + 3
        slots = torch.randperm(pages * page, generator=g, device=dev)[:t]
        if t > 1:
            slots[t // 2] = -1  # a token that has no slot: padding
        x = torch.randn(t, (4 if case["fused"] else 2) * h, DIM, generator=g, device=dev).to(dt)
        k, v = x[:, -2 * h:-h], x[:, -h:]
        if not case["fused"]:
            k, v = k.contiguous(), v.contiguous()
        pool = [_pool(pages, case, lambda *s: torch.zeros(s, dtype=dt, device=dev))
                for _ in range(2)]
        return dict(case=case, k=k, v=v, slots=slots, k_pages=pool[0], v_pages=pool[1],
                    error=torch.zeros(1, dtype=torch.int32, device=dev))

    before, new = _lengths(case)
    page, n = case["page"], case["requests"]
    total = sum(max(0, x) for x in new)
    held = [_pages(b if case["op"] == "step" else b + x, page) for b, x in zip(before, new)]
    width = max(_pages(b + max(0, x), page) for b, x in zip(before, new))
    pages = sum(_pages(b + max(0, x), page) for b, x in zip(before, new)) + 5
    ids = torch.randperm(pages, generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    held_t = torch.tensor(held, device=dev)
    start = torch.cumsum(held_t, 0) - held_t
    col = torch.arange(width, device=dev)
    table = torch.where(col < held_t[:, None],
                        ids[(start[:, None] + col).clamp(max=pages - 1)], -1).contiguous()
    i32 = dict(dtype=torch.int32, device=dev)
    if case["op"] == "step":
        free = sum(held)
        stack = torch.full((pages,), -1, **i32)
        stack[:pages - free] = ids[free:]
        return dict(case=case, lens=torch.tensor(before, **i32), new=torch.tensor(new, **i32),
                    table=table, stack=stack, count=torch.tensor([pages - free], **i32),
                    kv_lens=torch.zeros(n, **i32), cu_q=torch.zeros(n + 1, **i32),
                    slots=torch.zeros(total + 3, dtype=torch.int64, device=dev),
                    positions=torch.zeros(total + 3, **i32), count_out=torch.zeros(1, **i32),
                    error=torch.zeros(1, **i32))

    dt = DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(s, generator=g, device=dev, dtype=torch.float32).to(dt)  # noqa: E731
    k_pages, v_pages = _pool(pages, case, normal), _pool(pages, case, normal)
    # a few channels of K are much larger than the others, as in real models
    loud = torch.exp(torch.randn(4, generator=g, device=dev))
    k_pages[..., torch.randperm(DIM, generator=g, device=dev)[:4]] *= loud.to(dt)
    q = normal(total, case["q_heads"], DIM)
    cu = torch.zeros(n + 1, **i32)
    cu[1:] = torch.cumsum(torch.tensor(new, device=dev), 0)
    return dict(case=case, q=q, k_pages=k_pages, v_pages=v_pages, table=table, cu_q=cu,
                kv_lens=torch.tensor([b + x for b, x in zip(before, new)], **i32),
                max_q=max(new), max_kv=max(b + x for b, x in zip(before, new)),
                error=torch.zeros(1, **i32))


# --------------------------------------------------------------------- run --

def run(s):
    op = s["case"]["op"]
    if op == "step":
        if own:
            _ops().paged_step(s["lens"], s["new"], s["table"], s["stack"], s["count"],
                              page_size=s["case"]["page"], kv_lens=s["kv_lens"], cu_q=s["cu_q"],
                              slots=s["slots"], positions=s["positions"],
                              free_count_out=s["count_out"], error_flag=s["error"])
        else:
            _plain_step(s)
        return {k: s[k] for k in ("table", "stack", "kv_lens", "cu_q", "slots", "positions",
                                  "count_out", "error")}
    if op == "write":
        if own:
            _ops().paged_write(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"],
                               error_flag=s["error"])
        else:
            _plain_write(s)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if own:
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=s["q"].device)
        out = _ops().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu_q"],
                                     s["kv_lens"], max_q_len=s["max_q"], max_kv_len=s["max_kv"],
                                     window=s["case"]["window"], lse=lse,
                                     error_flag=s["error"])
        return {"out": out, "lse": lse}
    out, lse = _plain_attention(s)
    return {"out": out, "lse": lse}


def _plain_step(s):
    page, table, stack = s["case"]["page"], s["table"], s["stack"]
    lens, new = s["lens"].long(), s["new"].long()
    width = table.shape[1]
    done = new < 0
    add = torch.where(done, 0, new)
    have = (lens + page - 1) // page
    col = torch.arange(width, device=lens.device)
    # pages of ended requests go back on the stack
    back = torch.where(done, have, 0)
    count = s["count"].long()
    at = (count + torch.cumsum(back, 0) - back)[:, None] + col
    give = col < back[:, None]
    stack[at[give]] = table[give]
    top = count + back.sum()
    # pages that the new tokens need come off it, in request order
    need = torch.where(done, 0, (lens + add + page - 1) // page - have)
    wide = have + need > width
    need = torch.where(wide, 0, need)
    end = torch.cumsum(need, 0)
    served = ~wide & ((need == 0) | (end <= top))
    take = torch.where(served, need, 0)
    step = col - have[:, None]
    takes = (step >= 0) & (step < take[:, None])
    table[takes] = stack[(top - 1 - (end - need)[:, None] - step)[takes]]
    s["count_out"].copy_(top - take.sum())
    s["kv_lens"].copy_(torch.where(done, 0, torch.where(served, lens + add, lens)))
    s["cu_q"][1:] = torch.cumsum(add, 0)
    # where each new token goes
    token = torch.arange(s["slots"].numel(), device=lens.device)
    ends = s["cu_q"][1:].long()
    b = torch.searchsorted(ends, token, right=True).clamp(max=len(lens) - 1)
    position = lens[b] + token - (ends - add)[b]
    real = token < ends[-1]
    slot = table[b, (position // page).clamp(0, width - 1)].long() * page + position % page
    s["slots"].copy_(torch.where(real & served[b], slot, -1))
    s["positions"].copy_(torch.where(real, position, 0))
    s["error"].copy_((~served).any().int() * 3)


def _plain_write(s):
    page, keep = s["case"]["page"], s["slots"] >= 0
    slots = s["slots"][keep]
    for pool, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
        pool[slots // page, :, slots % page] = new[keep]


def _plain_attention(s):
    case, q = s["case"], s["q"]
    r, hk = case["q_heads"] // case["kv_heads"], case["kv_heads"]
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    n, mq, mk, t = len(kv), s["max_q"], s["max_kv"], q.shape[0]
    j = torch.arange(mk, device=q.device)
    page = s["table"][:, j // case["page"]].long().clamp(min=0)
    row = j % case["page"]
    # [n, mk, hk, D] rows of every request, in 32 bits
    held = (j < kv[:, None])[..., None, None]
    k = s["k_pages"][page, :, row].float()
    v = torch.where(held, s["v_pages"][page, :, row], 0).float()
    i = torch.arange(mq, device=q.device)
    q_len = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + i).clamp(max=t - 1)
    x = q[at].float().view(n, mq, hk, r, DIM).permute(0, 2, 1, 3, 4).reshape(n, hk, mq * r, DIM)
    score = torch.matmul(x, k.permute(0, 2, 3, 1)).view(n, hk, mq, r, mk)
    score.mul_(1.0 / math.sqrt(DIM))
    p = (kv - q_len)[:, None] + i
    seen = j <= p[..., None]
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(n, hk, mq * r, mk), v.permute(0, 2, 1, 3))
    out = out.view(n, hk, mq, r, DIM) / torch.where(total == 0, 1, total)
    lse = (top + torch.log(total))[..., 0]
    # back to one row per token
    token = torch.arange(t, device=q.device)
    b = torch.searchsorted(cu[1:], token, right=True).clamp(max=n - 1)
    i = token - cu[b]
    out = out.permute(0, 2, 1, 3, 4)[b, i].reshape(t, hk * r, DIM)
    return out.to(q.dtype), lse.permute(0, 2, 1, 3)[b, i].reshape(t, hk * r)


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    """Attention in 64 bits, request by request; the other operators only move values."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
    before, new = _lengths(case)
    r, window = case["q_heads"] // case["kv_heads"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=s["q"].device)
    first = 0
    for b, (old, x) in enumerate(zip(before, new)):
        ids = s["table"][b, :_pages(old + x, case["page"])].long()
        for h in range(case["kv_heads"]):
            k = s["k_pages"][ids, h].reshape(-1, DIM)[:old + x].double()
            v = s["v_pages"][ids, h].reshape(-1, DIM)[:old + x].double()
            for c in range(0, x, 1024):
                end = min(x, c + 1024)
                low = max(0, old + c - window + 1) if window else 0
                high = old + end
                q = s["q"][first + c:first + end, h * r:(h + 1) * r].double()
                e = q @ k[low:high].T / math.sqrt(DIM)
                gap = (torch.arange(old + c, high, device=e.device)[:, None]
                       - torch.arange(low, high, device=e.device))
                hide = (gap < 0) | (gap >= window) if window else gap < 0
                e = e.masked_fill(hide[:, None], -math.inf)
                z = torch.logsumexp(e, -1)
                out[first + c:first + end, h * r:(h + 1) * r] = torch.exp(e - z[..., None]) @ v[low:high]
                lse[first + c:first + end, h * r:(h + 1) * r] = z
        first += x
    return {"out": out, "lse": lse}
