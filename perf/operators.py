"""Timed cases of the paged key-value cache: the step plan (block tables and slot maps), the append of
new keys and values, and the attention of the new tokens over the cache.

``run`` computes an operator in plain torch where ``own`` is false and through
``syncopate_b200.computation.paged`` where it is true.  Both work on what ``prepare`` makes.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_E4M3_MAX = 448.0


def listed():
    return [
        # A decode step of a small server: a few running requests take one token each.
        dict(name="plan_small", op="plan", requests=8, page=16, max_len=1000, new=1, ended=0, tokens=8),
        # A decode step of a full server: most requests take a token, some are idle, some have ended.
        dict(name="plan_decode", op="plan", requests=1021, page=64, max_len=16384, new=1, ended=40, tokens=1024),
        # A step that takes in many prompts at once, lengths ragged, slot map padded to its capacity.
        dict(name="plan_prompts", op="plan", requests=96, page=16, max_len=8192, new=1500, ended=5, tokens=81920),
        # The keys and values of one decode step.
        dict(name="append_step", op="append", tokens=16, heads=8, dim=128, page=16, dtype="bf16", cache="same"),
        # The keys and values of a batch of prompts (an odd number of tokens).
        dict(name="append_prompts", op="append", tokens=32749, heads=8, dim=128, page=64, dtype="bf16", cache="same"),
        # The same into an 8-bit cache with a scale for each head.
        dict(name="append_e4m3", op="append", tokens=16381, heads=8, dim=128, page=32, dtype="bf16", cache="e4m3"),
        # One user's chat: a single request, latency is all that counts.
        dict(name="attend_one", op="attend", requests=1, q_heads=32, kv_heads=8, dim=128, page=16, min_len=700,
             max_len=700, new=1, window=0, dtype="bf16", cache="same"),
        # An ordinary decode batch of ragged lengths.
        dict(name="attend_batch", op="attend", requests=61, q_heads=32, kv_heads=8, dim=128, page=16, min_len=90,
             max_len=5003, new=1, window=0, dtype="bf16", cache="same"),
        # One long document: the only work to split is the cache's length.
        dict(name="attend_long", op="attend", requests=1, q_heads=32, kv_heads=4, dim=128, page=64, min_len=131071,
             max_len=131071, new=1, window=0, dtype="bf16", cache="same"),
        # A full server: a batch whose cache is gigabytes.
        dict(name="attend_full", op="attend", requests=128, q_heads=64, kv_heads=8, dim=128, page=32, min_len=1024,
             max_len=12288, new=1, window=0, dtype="bf16", cache="same"),
        # The same server on an 8-bit cache.
        dict(name="attend_e4m3", op="attend", requests=96, q_heads=32, kv_heads=8, dim=128, page=64, min_len=300,
             max_len=12007, new=1, window=0, dtype="bf16", cache="e4m3"),
        # Several drafted tokens a request are verified at once, in half precision, under a sliding window,
        # with small heads and pages that are no power of two.
        dict(name="attend_drafts", op="attend", requests=45, q_heads=24, kv_heads=6, dim=64, page=24, min_len=17,
             max_len=9001, new=7, window=4000, dtype="f16", cache="same"),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "attend"])
    if op == "plan":
        requests = _log(rng, 1, 2048)
        new = _log(rng, 1, max(1, 81920 // requests))
        return dict(op=op, requests=requests, page=rng.choice([8, 16, 24, 32, 64, 128]), max_len=_log(rng, 16, 16384),
                    new=new, ended=rng.randint(0, requests // 4), tokens=requests * new + rng.randint(0, 63))
    if op == "append":
        heads, dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 32749 * 1024 // (heads * dim) if heads * dim > 1024 else 32749),
                    heads=heads, dim=dim, page=rng.choice([8, 16, 20, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]), cache=rng.choice(["same", "same", "e4m3"]))
    kv_heads, group, dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 2, 4, 5, 7, 8, 16]), rng.choice([64, 128, 256])
    new = rng.choice([1, 1, 1, 2, 4, 9])
    max_len = _log(rng, 32, 131071)
    most = 128 * 12288 * 8 * 128 // (max_len * kv_heads * dim * max(1, group * new // 8))
    return dict(op=op, requests=_log(rng, 1, max(1, min(256, most))), q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                page=rng.choice([8, 16, 24, 32, 64, 128]), min_len=_log(rng, new, max_len), max_len=max_len, new=new,
                window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]), dtype=rng.choice(["bf16", "bf16", "f16"]),
                cache=rng.choice(["same", "same", "e4m3"]))


# ------------------------------------------------------------------ what a case's requests look like
# Lengths follow from the case alone and the seed gives their order, so that the work of a case is
# the same for every seed.


def _spread(low, high, n):
    return [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def _plan_requests(case, rng=None):
    """(tokens cached, tokens to append; -1 = the request has ended) of every request."""
    n, new, ended = case["requests"], case["new"], case["ended"]
    lens = _spread(0, case["max_len"], n)
    add = [new if new == 1 else 1 + (i * 97) % new for i in range(n)]
    for i in range(ended):
        add[(i * 7919) % n] = -1
    if new == 1:
        for i in range(5, n, 11):  # idle this step
            add[i] = min(add[i], 0)
    pairs = list(zip(lens, add))
    if rng is not None:
        rng.shuffle(pairs)
    return [p[0] for p in pairs], [p[1] for p in pairs]


def _attend_requests(case, rng=None):
    """(tokens cached, new ones among them) of every request."""
    n, new = case["requests"], case["new"]
    lens = _spread(max(case["min_len"], new), case["max_len"], n)
    news = [1 + (i * 5) % new for i in range(n)]
    pairs = list(zip(lens, news))
    if rng is not None:
        rng.shuffle(pairs)
    return [p[0] for p in pairs], [p[1] for p in pairs]


def _pages(n, page):
    return -(-n // page)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=dict(case))

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    if case["op"] == "plan":
        page = case["page"]
        lens, add = _plan_requests(case, rng)
        width = max(_pages(n + max(a, 0), page) for n, a in zip(lens, add)) + 1
        held = [_pages(n, page) for n in lens]
        need = sum(_pages(n + a, page) - h for n, a, h in zip(lens, add, held) if a >= 0)
        pages = sum(held) + need + 17
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        at = torch.arange(width, device="cuda")[None, :] < _ints(held)[:, None]
        table[at] = order[: sum(held)]
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[: pages - sum(held)] = order[sum(held):]
        state.update(lens=_ints(lens), add=_ints(add), table=table, free=free, num_free=_ints([pages - sum(held)]),
                     slots=_ints([0] * case["tokens"]), positions=_ints([0] * case["tokens"]), starts=_ints([0] * (len(lens) + 1)),
                     lens_out=_ints([0] * len(lens)), num_free_out=_ints([0]))
    elif case["op"] == "append":
        T, H, D, page, dt = case["tokens"], case["heads"], case["dim"], case["page"], _TYPES[case["dtype"]]
        pages = _pages(T, page) + 3
        # Keys and values come as columns of one projection, as a model's layer makes them.
        rows = normal(T, 3 * H * D, dtype=dt)
        state.update(k=rows[:, H * D: 2 * H * D].view(T, H, D), v=rows[:, 2 * H * D:].view(T, H, D))
        perm = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(T, device="cuda")
        slots = (perm[at // page] * page + at % page).to(torch.int32)
        slots[torch.rand(T, generator=gen, device="cuda") < 1 / 64] = -1  # padding rows of the batch
        state.update(slots=slots)
        if case["cache"] == "e4m3":
            for n in ("k", "v"):
                state[n + "_scale"] = torch.rand(H, generator=gen, device="cuda") * 0.01 + 0.004
                state[n + "_cache"] = normal(pages, page, H, D, scale=80.0).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
        else:
            state.update(k_cache=normal(pages, page, H, D, dtype=dt), v_cache=normal(pages, page, H, D, dtype=dt))
    else:
        Hq, H, D, page, dt = case["q_heads"], case["kv_heads"], case["dim"], case["page"], _TYPES[case["dtype"]]
        lens, news = _attend_requests(case, rng)
        held = [_pages(n, page) for n in lens]
        pages, T = sum(held) + 5, sum(news)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(lens), max(held)), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(max(held), device="cuda")[None, :] < _ints(held)[:, None]] = order[: sum(held)]
        state.update(q=normal(T, Hq, D, dtype=dt), table=table, lens=_ints(lens), out=torch.empty(T, Hq, D, dtype=dt, device="cuda"),
                     lse=torch.empty(T, Hq, device="cuda"))
        if case["new"] > 1:
            starts = [0]
            for n in news:
                starts.append(starts[-1] + n)
            state.update(starts=_ints(starts))
        kept = torch.float8_e4m3fn if case["cache"] == "e4m3" else dt
        for n in ("k", "v"):
            cache = torch.empty(pages, page, H, D, dtype=kept, device="cuda")
            for i in range(0, pages, 4096):  # a piece at a time: the 32-bit normals are larger than the cache
                part = cache[i: i + 4096]
                part.copy_(normal(*part.shape, scale=80.0 if kept != dt else 1.0).clamp_(-_E4M3_MAX, _E4M3_MAX))
            state[n + "_cache"] = cache
            if kept != dt:
                state[n + "_scale"] = torch.rand(H, generator=gen, device="cuda") * 0.01 + 0.008
    return state


# ------------------------------------------------------------------ plain forms


def _gather(x, at):
    # 8-bit floats are indexed as bytes.
    return x.view(torch.uint8)[at].view(x.dtype) if x.element_size() == 1 else x[at]


def _plain_plan(s):
    page, lens, add, table, free = s["case"]["page"], s["lens"].long(), s["add"].long(), s["table"], s["free"]
    held = (lens + page - 1) // page
    ended, more = add < 0, add.clamp(min=0)
    # Pages of ended requests go back onto the stack, in the order of the requests.
    given = torch.where(ended, held, 0)
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    back = column < given[:, None]
    top = s["num_free"].long()
    place = (top + given.cumsum(0) - given)[:, None] + column
    free[place[back]] = table[back]
    top = top + given.sum()
    # New pages come off its top, in the order of the requests.
    total = torch.where(ended, 0, lens + more)
    want = torch.where(ended, 0, (total + page - 1) // page - held)
    before = want.cumsum(0) - want
    fresh = (column >= held[:, None]) & (column < (held + want)[:, None])
    place = top - 1 - (before - held)[:, None] - column
    table[fresh] = free[place[fresh]]
    ends = more.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    at = torch.arange(s["slots"].numel(), device=table.device)
    z = torch.searchsorted(ends, at, right=True)
    live = z < lens.numel()
    z = z.clamp(max=lens.numel() - 1)
    position = lens[z] + at - starts[z]
    there = table[z, (position // page).clamp(0, table.shape[1] - 1)].long()
    slots = torch.where(live, there * page + position % page, -1)
    positions = torch.where(live, position, 0)
    i32 = torch.int32
    return slots.to(i32), positions.to(i32), starts.to(i32), total.to(i32), (top - want.sum()).to(i32), table, free


def _plain_append(s):
    page = s["case"]["page"]
    slots = s["slots"].long()
    live = slots >= 0
    at = slots[live]
    for n in ("k", "v"):
        cache, x = s[n + "_cache"], s[n][live]
        if s["case"]["cache"] == "e4m3":
            x = (x.float() / s[n + "_scale"][None, :, None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
            cache.view(torch.uint8)[at // page, at % page] = x.view(torch.uint8)
        else:
            cache[at // page, at % page] = x
    return s["k_cache"], s["v_cache"]


def _plain_attend(s):
    case = s["case"]
    page, H, D, window = case["page"], case["kv_heads"], case["dim"], case["window"]
    group, q, lens, table = case["q_heads"] // H, s["q"], s["lens"].long(), s["table"].long()
    T, Z, L = q.shape[0], lens.numel(), case["max_len"]
    key = torch.arange(L, device=q.device)
    at = table[:, key // page].clamp(min=0)  # [Z, L]
    k, v = (_gather(s[n + "_cache"].permute(2, 0, 1, 3), (slice(None), at, (key % page)[None, :])).float() for n in ("k", "v"))
    if case["cache"] == "e4m3":  # [H, Z, L, D]
        k, v = k.mul_(s["k_scale"].view(H, 1, 1, 1)), v.mul_(s["v_scale"].view(H, 1, 1, 1))
    new = case["new"]
    if new > 1:
        starts = s["starts"].long()
        count = starts[1:] - starts[:-1]
        i = torch.arange(new, device=q.device)
        real = i[None, :] < count[:, None]
        row = (starts[:-1, None] + i).clamp(max=T - 1)
    else:
        count, i = torch.ones_like(lens), torch.zeros(1, dtype=torch.long, device=q.device)
        real = torch.ones(Z, 1, dtype=torch.bool, device=q.device)
        row = torch.arange(Z, device=q.device)[:, None]
    rows = q.float()[row].view(Z, new, H, group, D).permute(2, 0, 1, 3, 4).reshape(H, Z, new * group, D)
    scores = torch.matmul(rows, k.transpose(2, 3)) * D ** -0.5
    position = (lens - count)[:, None] + i  # of each new token
    seen = (key <= position[..., None]) & (key < lens[:, None, None])
    if window:
        seen &= key > position[..., None] - window
    scores = scores.view(H, Z, new, group, L).masked_fill_(~seen[None, :, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(H, Z, new * group, L), v).view(H, Z, new, group, D) / total.clamp(min=1e-38)
    lse = (top + total.log()) / math.log(2.0)
    o = o.permute(1, 2, 0, 3, 4).reshape(Z, new, H * group, D)[real]
    return o.to(q.dtype), lse.permute(1, 2, 0, 3, 4).reshape(Z, new, H * group)[real]


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](s)
    from syncopate_b200.computation.paged import page_plan, paged_append, paged_attention

    if op == "plan":
        page_plan(s["lens"], s["add"], s["table"], s["free"], s["num_free"], s["case"]["page"], s["slots"], s["positions"],
                  s["starts"], lens_out=s["lens_out"], num_free_out=s["num_free_out"])
        return s["slots"], s["positions"], s["starts"], s["lens_out"], s["num_free_out"], s["table"], s["free"]
    if op == "append":
        paged_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], k_scale=s.get("k_scale"), v_scale=s.get("v_scale"))
        return s["k_cache"], s["v_cache"]
    paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["case"]["dim"] ** -0.5, starts=s.get("starts"),
                    window=s["case"]["window"], k_scale=s.get("k_scale"), v_scale=s.get("v_scale"), out=s["out"], lse=s["lse"])
    return s["out"], s["lse"]


# ------------------------------------------------------------------ work


def _spans(case):
    """(keys that some new token of the request sees, pairs of new token and key) of every request."""
    for length, new in zip(*_attend_requests(case)):
        window = case["window"] or length
        seen = [min(window, length - new + i + 1) for i in range(new)]
        yield length - max(0, length - new + 1 - window), sum(seen)


def work(case):
    if case["op"] == "plan":
        lens, add = _plan_requests(case)
        page = case["page"]
        moved = sum(_pages(n, page) if a < 0 else _pages(n + a, page) - _pages(n, page) for n, a in zip(lens, add))
        # Lengths and counts in, lengths and starts out; a page number is read and written for each page
        # that moves; slots and positions out; the page that each request's first new token falls into.
        return {"bytes": 4 * (5 * len(lens) + 2 * moved + 2 * case["tokens"] + 3), "flops": 0}
    if case["op"] == "append":
        item = 1 if case["cache"] == "e4m3" else 2
        return {"bytes": case["tokens"] * (4 + 2 * case["heads"] * case["dim"] * (2 + item) * 63 / 64), "flops": 0}
    item = 1 if case["cache"] == "e4m3" else 2
    lens, news = _attend_requests(case)
    spans = list(_spans(case))
    rows, D = sum(news) * case["q_heads"], case["dim"]
    keys = sum(n for n, _ in spans)
    return {"bytes": keys * case["kv_heads"] * D * 2 * item + rows * (4 * D + 4) + 4 * (len(lens) + keys // case["page"]),
            "flops": 4 * D * case["q_heads"] * sum(n for _, n in spans)}


# ------------------------------------------------------------------ 64 bits


def _exact_plan(s):
    page = s["case"]["page"]
    lens, add, table = s["lens"].tolist(), s["add"].tolist(), s["table"].tolist()
    free, top = s["free"].tolist(), int(s["num_free"])
    out_lens, starts, slots, positions = list(lens), [0], [], []
    for z, a in enumerate(add):
        if a < 0:
            for j in range(_pages(lens[z], page)):
                free[top] = table[z][j]
                top += 1
            out_lens[z] = 0
    for z, a in enumerate(add):
        for t in range(max(a, 0)):
            at = out_lens[z]
            if at % page == 0:
                top -= 1
                table[z][at // page] = free[top]
            slots.append(table[z][at // page] * page + at % page)
            positions.append(at)
            out_lens[z] += 1
        starts.append(len(slots))
    pad = s["slots"].numel() - len(slots)
    return tuple(torch.tensor(x, dtype=torch.int32) for x in
                 (slots + [-1] * pad, positions + [0] * pad, starts, out_lens, [top], table, free))


def _exact_append(s):
    page, both = s["case"]["page"], []
    for n in ("k", "v"):
        x, kept = s[n].double(), s[n + "_cache"].to(torch.float64)
        if s["case"]["cache"] == "e4m3":
            x = torch.clamp(x / s[n + "_scale"].double().view(1, -1, 1), -_E4M3_MAX, _E4M3_MAX)
        flat = kept.view(-1, *kept.shape[2:])
        rows = torch.nonzero(s["slots"] >= 0).view(-1)
        flat[s["slots"][rows].long()] = x[rows]
        both.append(flat.view(kept.shape))
    return tuple(both)


def _exact_attend(s):
    case, q = s["case"], s["q"].double()
    page, H, D = case["page"], case["kv_heads"], case["dim"]
    group = case["q_heads"] // H
    starts = s["starts"].tolist() if case["new"] > 1 else list(range(len(s["lens"]) + 1))
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for z, length in enumerate(s["lens"].tolist()):
        held = s["table"][z, : _pages(length, page)].long()
        k, v = (_gather(s[n + "_cache"], held).view(-1, H, D)[:length].to(torch.float64) for n in ("k", "v"))
        if case["cache"] == "e4m3":
            k, v = k * s["k_scale"].double()[None, :, None], v * s["v_scale"].double()[None, :, None]
        n = starts[z + 1] - starts[z]
        for i in range(n):
            last = length - n + i
            first = max(0, last - case["window"] + 1) if case["window"] else 0
            rows = q[starts[z] + i].view(H, group, D)
            x = torch.einsum("hgd,lhd->hgl", rows, k[first: last + 1]) / math.sqrt(D)
            norm = torch.logsumexp(x, -1, keepdim=True)
            out[starts[z] + i] = torch.einsum("hgl,lhd->hgd", torch.exp(x - norm), v[first: last + 1]).reshape(H * group, D)
            lse[starts[z] + i] = norm.reshape(-1) / math.log(2.0)
    return out, lse


def exact(case, seed):
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend}[case["op"]](prepare(case, seed))
