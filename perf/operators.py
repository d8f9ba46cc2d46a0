"""Cases for the paged KV cache operators: planning a step, appending to the pages, and attention through them.

A step of a server that holds requests of different lengths is `paged_plan` (which pages and slots the new tokens get),
`paged_rope_append` (rotate q and k, write k and v into their slots) and `sdpa_paged` (attention of the new tokens over
their request's pages). Head layouts are those of this repository's configurations: 32 query / 8 kv heads of 64 (the 1B
config), 12 / 12 heads of 64 (the 125M config), 8 / 2 heads of 16 (the small decode-test config). Everything is F32;
ids, lengths and positions are integral F32 values, as the framework's decode operators take them.
"""
import math
import random

import torch

own = False  # set by the caller: False computes the plain forms, True calls the framework's operators

DEV = "cuda"
ROPE_THETA = 10000.0
HEADS = [(32, 8, 64), (12, 12, 64), (8, 2, 16)]  # query heads, kv heads, head dim


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 8 conversations: every request gets one token, some of them a page
        {"name": "plan 8 decode", "op": "plan", "n": 8, "page": 16, "cached": 500, "chunk": 1, "mixed": False, "ended": False, "shape_seed": 1},
        # a large server's step: 1000 requests, most decode one token, some prefill a chunk, some have ended
        {"name": "plan 1000 mixed", "op": "plan", "n": 1000, "page": 16, "cached": 4000, "chunk": 256, "mixed": True, "ended": True, "shape_seed": 2},
        # decode step of 32 requests, 1B heads: 32 rows
        {"name": "append 32 decode", "op": "append", "n": 32, "page": 16, "cached": 2000, "chunk": 1, "mixed": False, "heads": 0, "pad": 0, "shape_seed": 3},
        # prompt chunks, 1B heads: about 8,000 rows
        {"name": "append chunks", "op": "append", "n": 16, "page": 16, "cached": 1000, "chunk": 1000, "mixed": False, "heads": 0, "pad": 0, "shape_seed": 4},
        # pages that are no power of two, 12 heads without groups, rows behind the last request
        {"name": "append odd", "op": "append", "n": 7, "page": 24, "cached": 333, "chunk": 201, "mixed": True, "heads": 1, "pad": 37, "shape_seed": 5},
        # one request decodes: latency
        {"name": "attend 1 decode", "op": "attend", "n": 1, "page": 16, "cached": 517, "chunk": 1, "mixed": False, "heads": 1, "pad": 0, "shape_seed": 6},
        # a decode step of 32 requests of different lengths
        {"name": "attend 32 decode", "op": "attend", "n": 32, "page": 16, "cached": 4096, "chunk": 1, "mixed": False, "heads": 0, "pad": 0, "shape_seed": 7},
        # four long contexts decode
        {"name": "attend long decode", "op": "attend", "n": 4, "page": 64, "cached": 60000, "chunk": 1, "mixed": False, "heads": 0, "pad": 0, "shape_seed": 8},
        # a few drafted tokens verified at once: more rows per kv head than a decode step, fewer than a tile
        {"name": "attend 6 new of 16", "op": "attend", "n": 16, "page": 16, "cached": 2500, "chunk": 6, "mixed": False, "heads": 0, "pad": 0, "shape_seed": 9},
        # one prompt chunk among decoding requests, rows behind the last request
        {"name": "attend mixed", "op": "attend", "n": 9, "page": 16, "cached": 4000, "chunk": 512, "mixed": True, "heads": 0, "pad": 24, "shape_seed": 10},
        # prompt chunks of about 2,000 tokens over cached prefixes
        {"name": "attend prefill", "op": "attend", "n": 4, "page": 16, "cached": 2048, "chunk": 2048, "mixed": False, "heads": 0, "pad": 0, "shape_seed": 11},
        # small heads, pages of 5 positions, odd lengths
        {"name": "attend small heads", "op": "attend", "n": 5, "page": 5, "cached": 777, "chunk": 131, "mixed": False, "heads": 2, "pad": 3, "shape_seed": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend"])
    while True:
        page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 128])
        case = {"op": op, "page": page, "shape_seed": rng.randrange(1 << 30)}
        if op == "plan":
            case |= {"n": _log(rng, 1, 1000), "cached": _log(rng, 1, 4000), "chunk": _log(rng, 1, 256), "mixed": rng.random() < 0.5, "ended": rng.random() < 0.5}
            if case["n"] * (case["cached"] + case["chunk"]) / page > 4_000_000:
                continue
        else:
            case |= {"heads": rng.choice([0, 0, 1, 2]), "pad": rng.choice([0, 0, 1, 50]), "mixed": rng.random() < 0.3}
            if op == "append":
                case |= {"n": _log(rng, 1, 64), "cached": _log(rng, 1, 2000), "chunk": _log(rng, 1, 1000)}
                if case["n"] * case["chunk"] > 16_000:
                    continue
            else:
                decode = rng.random() < 0.5
                case |= {"n": _log(rng, 1, 64), "cached": _log(rng, 1, 60000), "chunk": rng.choice([1, 1, 2, 3]) if decode else _log(rng, 4, 2048)}
        if op == "attend":
            h, kvh, d = HEADS[case["heads"]]
            most = case["cached"] + case["chunk"]
            if case["n"] * h * case["chunk"] * most > 4 * 32 * 2048 * 4096 or case["n"] * most * kvh * d > 4 * 60000 * 8 * 64:
                continue
        return case


def _shape(case):
    """Cached and new tokens of each request (a matter of the case, not of the seed)."""
    rng = random.Random(case["shape_seed"])
    cached, new = [], []
    for i in range(case["n"]):
        cached.append(rng.randint(case["cached"] // 2, case["cached"]))
        if case["mixed"]:  # one request in eight brings a chunk, the others decode
            new.append(rng.randint(max(1, case["chunk"] // 2), case["chunk"]) if i % 8 == 0 else 1)
        else:
            new.append(case["chunk"] if case["chunk"] <= 8 else rng.randint(max(1, case["chunk"] * 3 // 4), case["chunk"]))
        if case.get("ended") and i % 16 == 15:
            new[-1] = -1
    return cached, new


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    cached, new = _shape(case)
    p, rows = case["page"], sum(max(0, x) for x in new) + case.get("pad", 0)
    if case["op"] == "plan":
        need = sum(max(0, _pages(c + x, p) - _pages(c, p)) for c, x in zip(cached, new) if x >= 0)
        gone = sum(_pages(c, p) for c, x in zip(cached, new) if x < 0)
        touched = sum(_pages(c + x, p) - c // p for c, x in zip(cached, new) if x > 0)  # pages the new tokens lie in
        n = case["n"]
        return {"bytes": 4 * (2 * n + touched + need + 2 * gone + need + (n + 1) + n + 2 * rows + 4), "flops": 0}
    h, kvh, d = HEADS[case["heads"]]
    if case["op"] == "append":
        return {"bytes": 4 * rows * (2 * (h + 2 * kvh) * d + 2) + 8 * d * min(rows, max(c + x for c, x in zip(cached, new))),
                "flops": 3 * rows * (h + kvh) * d}
    keys = sum(c + x for c, x in zip(cached, new))
    pairs = sum(x * c + x * (x + 1) // 2 for c, x in zip(cached, new))
    return {"bytes": 4 * (2 * rows * h * d + 2 * keys * kvh * d + sum(_pages(c + x, p) for c, x in zip(cached, new)) + 2 * len(new) + 1),
            "flops": 4 * d * h * pairs}


# ---------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The step's tensors on the GPU, by name, and the numbers that a serving program knows on the host."""
    g = torch.Generator(device=DEV).manual_seed(seed * 1_000_003 + case["shape_seed"])
    cached, new = _shape(case)
    n, p = case["n"], case["page"]
    total = [c + x if x >= 0 else 0 for c, x in zip(cached, new)]
    held = [_pages(c, p) for c in cached]
    rows = sum(max(0, x) for x in new) + case.get("pad", 0)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    num = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
    host = {"page": p, "rows": rows, "max_new": max(1, max(new)), "max_len": max(total)}
    if case["op"] == "plan":
        # the pages held before the step are the first of a shuffled list; the others are free and stand in the ring
        free = sum(max(0, _pages(t, p) - h) for t, h, x in zip(total, held, new) if x >= 0) + n + 3
        order = torch.randperm(sum(held) + free, device=DEV, generator=g).float()
        wide = max(max(held), max(_pages(t, p) for t in total)) + 2
        col = torch.arange(wide, device=DEV)[None]
        hold = num(held).long()[:, None]
        first = hold.cumsum(0) - hold
        table = torch.where(col < hold, order[(first + col).clamp(max=order.numel() - 1)], -1.0)
        head = int(torch.randint(0, order.numel(), (1,), device=DEV, generator=g))
        ring = torch.full_like(order, -1.0)
        ring[(torch.arange(free, device=DEV) + head) % order.numel()] = order[sum(held):]
        return {"lengths": num(cached), "new": num(new), "table": table, "ring": ring, "state": num([head, free])}, host
    h, kvh, d = HEADS[case["heads"]]
    pages = [_pages(t, p) for t in total]
    blocks = sum(pages) + 5
    order = torch.randperm(blocks, device=DEV, generator=g)
    wide = max(pages) + 1
    col = torch.arange(wide, device=DEV)[None]
    hold = torch.tensor(pages, device=DEV)[:, None]
    first = hold.cumsum(0) - hold
    table = torch.where(col < hold, order[(first + col).clamp(max=blocks - 1)], -1)
    t = {"k_cache": rand(blocks, kvh, p, d), "v_cache": rand(blocks, kvh, p, d)}
    start = torch.tensor([0] + new, device=DEV).cumsum(0)
    qkv = rand(rows, (h + 2 * kvh) * d)  # the q | k | v product of the step's rows
    if case["op"] == "append":
        r = torch.arange(rows, device=DEV)
        req = torch.searchsorted(start[1:].contiguous(), r, right=True).clamp(max=n - 1)
        live = r < start[-1]
        pos = torch.where(live, torch.tensor(cached, device=DEV)[req] + r - start[req], 0)
        slots = torch.where(live, table[req, (pos // p).clamp(max=wide - 1)] * p + pos % p, -1)
        freq = ROPE_THETA ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        ang = torch.arange(host["max_len"], device=DEV, dtype=torch.float64)[:, None] * freq
        ang = torch.cat([ang, ang], 1)
        return t | {"qkv": qkv, "cos": ang.cos().float(), "sin": ang.sin().float(), "slots": slots.float(), "positions": pos.float()}, host
    return t | {"qkv": qkv, "table": table.float(), "q_start": start.float(), "kv_len": num(total)}, host


class _Owned:
    """Framework tensors that one state holds; they go back to the backend with it."""

    def __init__(self, be):
        self.be, self.tensors = be, []

    def drop(self):
        for t in self.tensors:
            self.be.release(t)
        self.tensors = []

    def __del__(self):
        self.drop()


class _Cuda:
    """A framework tensor's memory under the CUDA array interface, keeping its owner."""

    def __init__(self, t, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": "<f4", "data": (t.base, False), "version": 3, "strides": None}


_shared = []


def _backend():
    if not _shared:
        import __graft_entry__

        _shared.append(__graft_entry__.load_package().cuda_backend(0))
    return _shared[0]


def prepare(case, seed):
    tensors, host = _inputs(case, seed)
    state = {"op": case["op"], "heads": HEADS[case["heads"]] if "heads" in case else None, "host": host}
    if own:
        # The framework's operators take tensors of its own allocator: the same values are put there.
        be = _backend()
        mine, made, views = _Owned(be), {}, {}
        for name, t in tensors.items():
            made[name] = be.allocate(tuple(t.shape))
            mine.tensors.append(made[name])
        be.sync()
        for name, t in tensors.items():
            views[name] = torch.as_tensor(_Cuda(made[name], mine), device=DEV)
            views[name].copy_(t)
        torch.cuda.synchronize()
        if "qkv" in made:
            # q, k and v are views of the fused product, as the model's attention has them
            from projectai_b200 import cabi

            h, kvh, d = state["heads"]
            whole, at = cabi.reshape(made["qkv"], (host["rows"], h + 2 * kvh, d)), 0
            for name, heads in (("q", h), ("k", kvh), ("v", kvh)):
                made[name] = cabi.slice_view(whole, 1, at, heads)
                at += heads
        return state | {"be": be, "pai": made, "mine": mine, "views": views, "results": _Owned(be), "seen": {}}
    return state | tensors


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan, "append": _append, "attend": _attend}[state["op"]](state)


def _run_own(state):
    be, t, host = state["be"], state["pai"], state["host"]
    state["results"].drop()  # the last pass's results
    if state["op"] == "plan":
        got = be.paged_plan(t["lengths"], t["new"], t["table"], t["ring"], t["state"], host["page"], host["rows"])
        named = zip(("q_start", "kv_len", "slots", "positions", "state"), got)
        kept = {k: state["views"][k] for k in ("table", "ring")}
    elif state["op"] == "append":
        named = [("q", be.paged_rope_append(t["q"], t["k"], t["v"], t["cos"], t["sin"], t["positions"], t["slots"], t["k_cache"], t["v_cache"]))]
        kept = {k: state["views"][k] for k in ("k_cache", "v_cache")}
    else:
        scale = 1.0 / math.sqrt(state["heads"][2])
        named = [("out", be.sdpa_paged(t["q"], t["k_cache"], t["v_cache"], t["table"], t["q_start"], t["kv_len"], scale, host["max_new"]))]
        kept = {}
    out = kept
    for name, r in named:
        state["results"].tensors.append(r)
        at = (r.base, r.shape)  # the allocator gives most passes the same block: its torch view is made once
        if at not in state["seen"]:
            state["seen"][at] = torch.as_tensor(_Cuda(r, state["results"]), device=DEV)
        out[name] = state["seen"][at]
    return out


# ---------------------------------------------------------------- plain forms
def _plan(s):
    p, rows = s["host"]["page"], s["host"]["rows"]
    length, new, ring, table = s["lengths"].long(), s["new"].long(), s["ring"], s["table"]
    n, wide, size = length.numel(), table.shape[1], ring.numel()
    head, count = s["state"].long()
    gone, add = new < 0, new.clamp(min=0)
    kv_len = torch.where(gone, 0, length + add)
    have = (length + p - 1) // p
    need = torch.where(gone, 0, (kv_len + p - 1) // p - have)
    free = torch.where(gone, have, 0)
    start = torch.zeros(n + 1, dtype=torch.long, device=DEV)
    start[1:] = add.cumsum(0)
    col = torch.arange(wide, device=DEV)[None]
    base = (need.cumsum(0) - need)[:, None]
    r = col - have[:, None]
    fresh = (r >= 0) & (r < need[:, None])
    pushed = torch.where(col < free[:, None], (head + count + (free.cumsum(0) - free)[:, None] + col) % size, size)
    table.copy_(torch.where(fresh, ring[(head + base + r) % size], table))
    ring.copy_(torch.cat([ring, ring[:1]]).index_put((pushed.reshape(-1),), table.reshape(-1))[:size])
    t = torch.arange(rows, device=DEV)
    req = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=n - 1)
    live = t < start[-1]
    pos = torch.where(live, length[req] + t - start[req], 0)
    slot = torch.where(live, table[req, (pos // p).clamp(max=wide - 1)].long() * p + pos % p, -1)
    left = torch.stack([(head + need.sum()) % size, count - need.sum() + free.sum()])
    return {"q_start": start.float(), "kv_len": kv_len.float(), "slots": slot.float(), "positions": pos.float(), "state": left.float(),
            "table": table, "ring": ring}


def _split(s, rows):
    h, kvh, d = s["heads"]
    whole = s["qkv"].view(rows, h + 2 * kvh, d)
    return whole[:, :h], whole[:, h:h + kvh], whole[:, h + kvh:]


def _append(s):
    p = s["host"]["page"]
    q, k, v = _split(s, s["host"]["rows"])
    pos, slot = s["positions"].long(), s["slots"].long()
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    half = q.shape[2] // 2

    def turned(x):
        return x * c + torch.cat([-x[..., half:], x[..., :half]], -1) * sn

    live = slot >= 0
    at = slot[live]
    s["k_cache"][at // p, :, at % p] = turned(k)[live]
    s["v_cache"][at // p, :, at % p] = v[live]
    return {"q": turned(q), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend(s):
    p, rows, most, longest = s["host"]["page"], s["host"]["rows"], s["host"]["max_new"], s["host"]["max_len"]
    h, kvh, d = s["heads"]
    q = _split(s, rows)[0]
    start, length = s["q_start"].long(), s["kv_len"].long()
    n, g, cols = length.numel(), h // kvh, _pages(longest, p)
    new = start[1:] - start[:-1]
    pages = s["table"][:, :cols].long().clamp(min=0)
    k = s["k_cache"][pages].permute(0, 2, 1, 3, 4).reshape(n, kvh, cols * p, d)
    v = s["v_cache"][pages].permute(0, 2, 1, 3, 4).reshape(n, kvh, cols * p, d)
    step = torch.arange(most, device=DEV)
    at = start[:-1, None] + step
    live = step < new[:, None]
    x = q[at.clamp(max=rows - 1)] * (1.0 / math.sqrt(d))  # [n, most, h, d]
    x = x.view(n, most, kvh, g, d).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * most, d)
    score = (x @ k.transpose(2, 3)).view(n, kvh, g, most, cols * p)
    pos = (length - new)[:, None] + step
    seen = torch.arange(cols * p, device=DEV) <= pos[..., None]  # [n, most, keys]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = score.view(n, kvh, g * most, cols * p) @ v
    o = (o.view(n, kvh, g, most, d) / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(n, most, h, d)
    out = torch.zeros(rows, h, d, device=DEV)
    out[at[live]] = o[live]
    return {"out": out}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    t, host = _inputs(case, seed)
    p, rows = host["page"], host["rows"]
    cached, new = _shape(case)
    if case["op"] == "plan":
        table, ring = t["table"].long().tolist(), t["ring"].long().tolist()
        head, count = t["state"].long().tolist()
        taken, back, start, kv, slots, positions = 0, [], [0], [], [], []
        for i, (c, x) in enumerate(zip(cached, new)):
            if x < 0:
                back += table[i][:_pages(c, p)]
            for j in range(_pages(c, p), _pages(c + x, p) if x > 0 else 0):
                table[i][j] = ring[(head + taken) % len(ring)]
                taken += 1
            for y in range(c, c + x):
                positions.append(y)
                slots.append(table[i][y // p] * p + y % p)
            start.append(start[-1] + max(0, x))
            kv.append(c + x if x >= 0 else 0)
        for j, page in enumerate(back):
            ring[(head + count + j) % len(ring)] = page
        pad = rows - len(slots)
        f = lambda v: torch.tensor(v, dtype=torch.float64)  # noqa: E731
        return {"q_start": f(start), "kv_len": f(kv), "slots": f(slots + [-1] * pad), "positions": f(positions + [0] * pad),
                "state": f([(head + taken) % len(ring), count - taken + len(back)]), "table": f(table), "ring": f(ring)}
    h, kvh, d = HEADS[case["heads"]]
    x = t["qkv"].double().view(rows, h + 2 * kvh, d)
    if case["op"] == "append":
        pos = t["positions"].long()
        c, s = t["cos"].double()[pos][:, None], t["sin"].double()[pos][:, None]
        a, b = x[:, :h + kvh, :d // 2], x[:, :h + kvh, d // 2:]
        y = torch.cat([a * c[..., :d // 2] - b * s[..., :d // 2], b * c[..., d // 2:] + a * s[..., d // 2:]], -1)
        out = {"q": y[:, :h], "k_cache": t["k_cache"].double(), "v_cache": t["v_cache"].double()}
        count = sum(new)
        at = t["slots"][:count].long()
        for name, rowsof in (("k_cache", y[:count, h:]), ("v_cache", x[:count, h + kvh:])):
            flat = out[name].permute(0, 2, 1, 3).reshape(-1, kvh, d)
            flat[at] = rowsof
            out[name] = flat.view(-1, p, kvh, d).permute(0, 2, 1, 3)
        return out
    out, at = torch.zeros(rows, h, d, dtype=torch.float64, device=DEV), 0
    for i, (c, y) in enumerate(zip(cached, new)):
        ids = t["table"][i, :_pages(c + y, p)].long()
        k, v = (t[name][ids].double().transpose(0, 1).reshape(kvh, -1, d)[:, :c + y] for name in ("k_cache", "v_cache"))
        late = torch.arange(c + y, device=DEV)[None] > torch.arange(c, c + y, device=DEV)[:, None]
        for j in range(h):
            w = (x[at:at + y, j] @ k[j // (h // kvh)].T / math.sqrt(d)).masked_fill_(late, -math.inf)
            out[at:at + y, j] = torch.softmax(w, -1) @ v[j // (h // kvh)]
        at += y
    return {"out": out}
