"""Attention that reads a part of its cache, as cases that can be timed and checked.

A decoder that attends to everything reads its whole cache for every token, and behind long contexts that is most of a
step.  Three operators let a row of a step read some pages of 64 tokens instead: ``page_bounds`` keeps, beside the
cache, the lowest and the highest value of every key channel of each page that is full; ``select_pages`` takes from
these bounds, for every row and key head, the pages whose keys could score highest; ``attention_pages`` attends to the
keys of the listed pages alone.  A case is one call of one of them for one layer (``page_bounds``: one call for all the
layers of a step of single tokens, as the engine makes it).  Head layouts are those of the named configurations.

``exact`` computes the same from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

PAGE = 64
DEVICE = "cuda:0"


def listed():
    return [
        # one token each of sixteen sequences, all layers of the 8B sizes: a few of the sequences fill a page
        {"name": "bounds-tokens-16", "work": "bounds", "dtype": "bfloat16", "planes": 36, "kv_heads": 8, "d": 128, "seqs": 16, "context": 1000, "new": 1},
        # prompts that start together, unequal, one layer
        {"name": "bounds-prompts-8", "work": "bounds", "dtype": "bfloat16", "planes": 1, "kv_heads": 8, "d": 128, "seqs": 8, "context": 0, "new": 2048},
        # a long document evaluated in passes of 16384 rows: a late pass
        {"name": "bounds-pass", "work": "bounds", "dtype": "bfloat16", "planes": 1, "kv_heads": 8, "d": 128, "seqs": 1, "context": 20011, "new": 16384},
        # one user's next token behind a long context: latency
        {"name": "select-token-1", "work": "select", "dtype": "bfloat16", "heads": 16, "kv_heads": 8, "d": 128, "seqs": 1, "context": 32768, "new": 1, "top": 32},
        # a busy server: an odd number of sequences of very different lengths
        {"name": "select-tokens-50", "work": "select", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128, "seqs": 50, "context": 40000, "new": 1, "top": 64},
        # the next portion of a long document
        {"name": "select-chunk", "work": "select", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128, "seqs": 1, "context": 30700, "new": 2000, "top": 32},
        # the 32-bit path: two turns with heads of 64
        {"name": "select-turns-f32", "work": "select", "dtype": "float32", "heads": 14, "kv_heads": 2, "d": 64, "seqs": 2, "context": 9000, "new": 37, "top": 24},
        # the tokens of the selections above
        {"name": "attend-token-1", "work": "attend", "dtype": "bfloat16", "heads": 16, "kv_heads": 8, "d": 128, "seqs": 1, "context": 32768, "new": 1, "top": 32},
        {"name": "attend-tokens-50", "work": "attend", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128, "seqs": 50, "context": 40000, "new": 1, "top": 64},
        # a chat's next turn, a short message behind a long context
        {"name": "attend-turn-90", "work": "attend", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128, "seqs": 1, "context": 20000, "new": 90, "top": 32},
        # the portion of the document; the most work of a call of this list
        {"name": "attend-chunk", "work": "attend", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "d": 128, "seqs": 1, "context": 30700, "new": 2000, "top": 32},
        # the 32-bit path's tokens
        {"name": "attend-tokens-3-f32", "work": "attend", "dtype": "float32", "heads": 16, "kv_heads": 8, "d": 128, "seqs": 3, "context": 9000, "new": 1, "top": 24},
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    most = {w: max(_cost(c) for c in listed() if c["work"] == w) for w in ("bounds", "select", "attend")}
    while True:
        work = rng.choice(["bounds", "select", "select", "attend", "attend"])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        case = {"work": work, "dtype": dtype}
        if work == "bounds":
            case["planes"] = rng.choice([1, 1, rng.randint(2, 36)])
        else:
            case["heads"] = 0
        case.update(kv_heads=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128, 128]), seqs=_log_int(rng, 1, 50), context=_log_int(rng, 30, 40000))
        case["new"] = rng.choice([1, 1, _log_int(rng, 2, 2000)])
        if work != "bounds":
            case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 4, 7, 8])
            case["top"] = _log_int(rng, 4, 64)
        if work == "select" and case["context"] < 2 * PAGE * case["top"]:
            continue      # a context that is read in full leaves nothing to select
        if work == "bounds" and case["new"] > 1 and case["context"] % PAGE + case["new"] < PAGE:
            continue      # no page is filled
        if case["seqs"] * (case["context"] + case["new"]) <= 1200000 and (case.get("planes", 1) - 1) * case["seqs"] * case["context"] <= 600000 and _cost(case) <= most[work]:
            return case


# ---- the inputs ---------------------------------------------------------------------------------------------
def _sequences(case):
    """(tokens before the call, rows in it) of every sequence: the longest as stated, the others spread below it."""
    r = random.Random(case["seqs"] * 1000003 + case["context"] * 7 + case["new"])
    out = [(case["context"], case["new"])]
    for _ in range(case["seqs"] - 1):
        past = _log_int(r, max(1, case["context"] // 16), case["context"]) if case["context"] else 0
        new = 1 if case["new"] == 1 else _log_int(r, max(1, case["new"] // 16), case["new"])
        out.append((past, new))
    if case["work"] == "bounds" and case["new"] == 1:
        # one in four fills its page with this token (in use one in 64 does, and most calls have nothing to do)
        out = [(past // PAGE * PAGE + 63 if i % 4 == 0 else past, new) for i, (past, new) in enumerate(out)]
    return out


def _dtype(case):
    return getattr(torch, case["dtype"])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 17)
    r = random.Random(seed)
    seqs, dt, kvh, d = _sequences(case), _dtype(case), case["kv_heads"], case["d"]

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)
    held = [(past + new + PAGE - 1) // PAGE for past, new in seqs]
    pages = sum(held) + 1
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros((len(seqs) + 3, max(held)), dtype=torch.int32, device=DEVICE)
    slots = r.sample(range(len(seqs) + 3), len(seqs))
    at, starts, row = 0, [], 0
    for slot, n, (_, new) in zip(slots, held, seqs):
        table[slot, :n] = order[at:at + n]
        at += n
        starts.append(row)
        row += new
    s = {"case": case, "table": table, "slot": ints(slots), "q_start": ints(starts), "q_len": ints([n for _, n in seqs]),
         "kv_len": ints([p + n for p, n in seqs]), "nseq": len(seqs), "max_q": max(n for _, n in seqs), "rows": row, "seqs": seqs, "slots": slots,
         "starts": starts, "scale": d ** -0.5}
    # Keys as norm and rotation leave them: of unit size, some channels with a mean of their own, the keys of a page
    # alike in part (a passage of the text has a topic).
    planes = case.get("planes", 1)
    topic = torch.randn((planes, pages, kvh, 1, d), generator=g, device=DEVICE) * 0.6
    keys = torch.empty((planes, pages, kvh, PAGE, d), dtype=dt, device=DEVICE)
    mean = torch.randn((kvh, 1, d), generator=g, device=DEVICE) * (torch.rand((kvh, 1, d), generator=g, device=DEVICE) < 0.1) * 1.5
    for plane in range(planes):
        for lo in range(0, pages, 1024):
            part = keys[plane, lo:lo + 1024]
            noise = torch.randn(part.shape, generator=g, device=DEVICE, dtype=dt)
            part.copy_(noise * 0.7 + topic[plane, lo:lo + 1024] + mean)
    if case["work"] == "bounds":
        s["keys"] = keys if planes > 1 else keys[0]
        s["bounds"] = torch.zeros(s["keys"].shape[:-2] + (2, d), dtype=dt, device=DEVICE)
        return s
    topic, keys = topic[0, :, :, 0], keys[0]
    bounds = torch.stack((keys.amin(2), keys.amax(2)), 2)
    heads = case["heads"]
    G = heads // kvh
    # Queries look for a few passages each, and rows that follow one another look for nearly the same ones.
    qkv = torch.empty((row, (heads + 2 * kvh) * d), dtype=dt, device=DEVICE)
    for i, (past, new) in enumerate(seqs):
        mine = table[slots[i], :held[i]].long()
        spans = (new + 39) // 40
        pick = mine[torch.randint(0, held[i], (spans, 5), generator=g, device=DEVICE)]
        want = topic[pick].sum(1).repeat_interleave(40, 0)[:new].unsqueeze(2)          # [new, kv heads, 1, d]
        q = torch.randn((new, kvh, G, d), generator=g, device=DEVICE) * 0.6 + want * 0.6
        qkv[starts[i]:starts[i] + new, :heads * d] = q.reshape(new, heads * d).to(dt)
    s["q"] = qkv[:, :heads * d]
    s["pages"] = torch.full((row, kvh, case["top"]), -1, dtype=torch.int32, device=DEVICE)
    if case["work"] == "select":
        s["bounds"] = bounds
        return s
    s["bounds"] = bounds
    s["pages"] = _select(s, torch.float32)
    del s["bounds"]
    s["keys"] = keys
    s["values"] = torch.empty_like(keys)
    for lo in range(0, pages, 1024):
        part = s["values"][lo:lo + 1024]
        part.copy_(torch.randn(part.shape, generator=g, device=DEVICE, dtype=dt))
    s["out"] = torch.zeros((row, heads * d), dtype=dt, device=DEVICE)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------
FIRST, LAST = 1, 2      # pages at the sequence's start and up to the row's own that are always read


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["work"] == "bounds":
        return _bounds(state)
    if case["work"] == "select":
        return _select(state, torch.float64)
    return _attend_tokens(state) if state["max_q"] == 1 else _attend_rows(state)


def _run_own(s):
    from gophonic_b200 import ops
    case = s["case"]
    if case["work"] == "bounds":
        ops.page_bounds(s["keys"], s["bounds"], s["table"], s["slot"], s["q_len"], s["kv_len"], s["nseq"], s["max_q"])
        return s["bounds"]
    if case["work"] == "select":
        ops.select_pages(s["q"], s["bounds"], s["table"], s["slot"], s["q_start"], s["q_len"], s["kv_len"], s["nseq"], s["max_q"],
                         case["heads"], case["kv_heads"], case["d"], s["pages"], FIRST, LAST)
        return s["pages"]
    ops.attention_pages(s["q"], s["out"], s["keys"], s["values"], s["table"], s["slot"], s["q_start"], s["q_len"], s["kv_len"], s["nseq"],
                        s["max_q"], case["heads"], case["kv_heads"], case["d"], s["scale"], s["pages"])
    return s["out"]


def _bounds(s):
    """The extremes of every key channel over the pages that this step's rows fill."""
    keys, bounds = (t if t.dim() == 5 else t.unsqueeze(0) for t in (s["keys"], s["bounds"]))
    for slot, (past, new) in zip(s["slots"], s["seqs"]):
        lo, hi = past // PAGE, (past + new) // PAGE
        if lo < hi:
            full = s["table"][slot, lo:hi].long()
            k = keys[:, full]
            bounds[:, full, :, 0] = k.amin(3)
            bounds[:, full, :, 1] = k.amax(3)
    return s["bounds"]


def _select(s, dtype):
    """Scores from the bounds, then the ``top`` pages of each row and key head: those always read, then the highest scores."""
    case = s["case"]
    kvh, d, top = case["kv_heads"], case["d"], case["top"]
    out = torch.empty_like(s["pages"])
    for slot, start, (past, new) in zip(s["slots"], s["starts"], s["seqs"]):
        held = (past + new + PAGE - 1) // PAGE
        b = s["bounds"][s["table"][slot, :held].long()].to(dtype)                        # [pages, kv heads, 2, d]
        low, high = b[:, :, 0].permute(1, 2, 0), b[:, :, 1].permute(1, 2, 0)             # [kv heads, d, pages]
        number = torch.arange(held, device=DEVICE)
        step = max(1, (1 << 25) // (kvh * held))
        for a in range(0, new, step):
            n = min(step, new - a)
            q = s["q"][start + a:start + a + n].reshape(n, kvh, -1, d).to(dtype)
            up, down = q.clamp(min=0).sum(2).transpose(0, 1), q.clamp(max=0).sum(2).transpose(0, 1)
            score = (up @ high + down @ low).transpose(0, 1)                             # [rows, kv heads, pages]
            score = torch.where(score.isnan(), -math.inf, score)
            last = ((past + a + torch.arange(n, device=DEVICE)) // PAGE).view(n, 1, 1)   # the page of the row itself
            kind = torch.where((number < FIRST) | (number > last - LAST), 0, 1)
            kind = torch.where(number > last, 2, kind).expand(n, kvh, held)
            by_score = score.sort(dim=-1, descending=True, stable=True).indices
            order = by_score.gather(-1, kind.gather(-1, by_score).sort(dim=-1, stable=True).indices)[..., :top]
            chosen = torch.where(kind.gather(-1, order) < 2, order, held).sort(dim=-1).values
            chosen = torch.where(chosen < held, chosen, -1)
            out[start + a:start + a + n] = -1
            out[start + a:start + a + n, :, :chosen.shape[-1]] = chosen.to(torch.int32)
    return out


def _attend_tokens(s):
    """Single tokens: the listed pages are gathered, one softmax over them."""
    case = s["case"]
    kvh, d = case["kv_heads"], case["d"]
    for i, (past, _) in enumerate(s["seqs"]):
        listed_ = s["pages"][i].long()                                                   # [kv heads, top]
        phys = s["table"][s["slots"][i]][listed_.clamp(min=0)].long()
        head = torch.arange(kvh, device=DEVICE).view(kvh, 1)
        k = s["keys"][phys, head].float().reshape(kvh, -1, d)
        v = s["values"][phys, head].float().reshape(kvh, -1, d)
        at = (listed_.unsqueeze(-1) * PAGE + torch.arange(PAGE, device=DEVICE)).reshape(kvh, 1, -1)
        seen = (at >= 0) & (at <= past)
        q = s["q"][i].float().reshape(kvh, -1, d)
        score = torch.where(seen, q @ k.transpose(1, 2) * s["scale"], -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        s["out"][i] = ((p / p.sum(-1, keepdim=True)) @ v).reshape(-1).to(s["out"].dtype)
    return s["out"]


def _attend_rows(s):
    """Rows of longer runs: scores over the whole context, masked to the listed pages."""
    case = s["case"]
    kvh, d = case["kv_heads"], case["d"]
    for slot, start, (past, new) in zip(s["slots"], s["starts"], s["seqs"]):
        held = (past + new + PAGE - 1) // PAGE
        phys = s["table"][slot, :held].long()
        k = s["keys"][phys].float().transpose(0, 1).reshape(kvh, 1, held * PAGE, d)
        v = s["values"][phys].float().transpose(0, 1).reshape(kvh, 1, held * PAGE, d)
        step = max(1, (1 << 28) // (case["heads"] * held * PAGE))
        for a in range(0, new, step):
            n = min(step, new - a)
            listed_ = s["pages"][start + a:start + a + n].long()                         # [rows, kv heads, top]
            use = torch.zeros((n, kvh, held + 1), dtype=torch.bool, device=DEVICE)
            use.scatter_(2, torch.where(listed_ < 0, held, listed_), True)
            here = past + a + torch.arange(n, device=DEVICE)
            seen = use[..., :held].repeat_interleave(PAGE, 2) & (torch.arange(held * PAGE, device=DEVICE) <= here.view(n, 1, 1))
            q = s["q"][start + a:start + a + n].float().reshape(n, kvh, -1, d).permute(1, 2, 0, 3)
            score = torch.where(seen.transpose(0, 1).unsqueeze(1), q @ k.transpose(2, 3) * s["scale"], -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            ctx = (p / p.sum(-1, keepdim=True)) @ v                                      # [kv heads, group, rows, d]
            s["out"][start + a:start + a + n] = ctx.permute(2, 0, 1, 3).reshape(n, -1).to(s["out"].dtype)
    return s["out"]


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def work(case):
    seqs, size = _sequences(case), 4 if case["dtype"] == "float32" else 2
    kvh, d = case["kv_heads"], case["d"]
    if case["work"] == "bounds":
        full = sum((past + new) // PAGE - past // PAGE for past, new in seqs) * case["planes"] * kvh
        return {"bytes": full * (PAGE + 2) * d * size + 12 * len(seqs), "flops": 2 * full * PAGE * d}
    heads, top = case["heads"], case["top"]
    rows = sum(new for _, new in seqs)
    if case["work"] == "select":
        held = sum((past + new) // PAGE for past, new in seqs)
        pairs = sum(new * ((past + new // 2) // PAGE) for past, new in seqs)
        return {"bytes": (held * kvh * 2 + rows * heads) * d * size + rows * kvh * top * 4, "flops": 4 * pairs * kvh * d}
    read = pairs = 0
    for past, new in seqs:
        held = (past + new + PAGE - 1) // PAGE
        # rows near one another read nearly the same pages; every page of the context at most once
        read += min(held, min(top, held) * ((new + 39) // 40))
        pairs += new * min(top, held) * PAGE
    return {"bytes": (read * kvh * 2 * PAGE + 2 * rows * heads) * d * size + rows * kvh * top * 4, "flops": 4 * pairs * heads * d}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / (6.0e13 if case["dtype"] == "float32" else 1.0e15)


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kvh, d = case["kv_heads"], case["d"]
    if case["work"] == "bounds":
        return _exact_bounds(s)
    rows = [(i, past + j, s["starts"][i] + j) for i, (past, new) in enumerate(s["seqs"]) for j in range(new)]
    if case["work"] == "select":
        pages = sum((pos // PAGE + 1) for _, pos, _ in rows)
        if pages * case["heads"] * d > 60e9 or len(rows) > 6000:
            return None
        return _exact_select(s)
    if len(rows) * kvh * case["top"] * PAGE * d > 30e9 or len(rows) > 6000:
        return None
    out = torch.zeros((s["rows"], case["heads"], d), dtype=torch.float64, device=DEVICE)
    for i, pos, row in rows:
        pages = s["pages"][row]
        table = s["table"][s["slots"][i]].long()
        where = pages.clamp(min=0).long()
        kv = [torch.stack([t[table[where[h]], h] for h in range(kvh)]).double().reshape(kvh, -1, d) for t in (s["keys"], s["values"])]
        token = (where.unsqueeze(2) * PAGE + torch.arange(PAGE, device=DEVICE)).reshape(kvh, -1)
        hidden = (pages < 0).repeat_interleave(PAGE, 1) | (token > pos)
        z = torch.einsum("hgd,htd->hgt", s["q"][row].double().reshape(kvh, -1, d), kv[0]) * s["scale"]
        z = z.masked_fill(hidden.unsqueeze(1), -math.inf)
        out[row] = torch.einsum("hgt,htd->hgd", torch.softmax(z, dim=-1), kv[1]).reshape(-1, d)
    return out.reshape(s["rows"], -1)


def _exact_bounds(s):
    out = s["bounds"].double()
    keys = s["keys"] if s["keys"].dim() == 5 else s["keys"].unsqueeze(0)
    planes = out if out.dim() == 5 else out.unsqueeze(0)
    for slot, (past, new) in zip(s["slots"], s["seqs"]):
        for page in range(max(0, past - 63) // PAGE, (past + new) // PAGE):
            if past < (page + 1) * PAGE <= past + new:
                p = int(s["table"][slot, page])
                ordered = keys[:, p].double().sort(dim=2).values
                planes[:, p] = torch.stack((ordered[:, :, 0], ordered[:, :, -1]), 2)
    return out


def _exact_select(s):
    case = s["case"]
    kvh, d, top = case["kv_heads"], case["d"], case["top"]
    out = torch.full_like(s["pages"], -1)
    for slot, start, (past, new) in zip(s["slots"], s["starts"], s["seqs"]):
        for j in range(new):
            mine = (past + j) // PAGE
            b = s["bounds"][s["table"][slot, :mine + 1].long()].double().unsqueeze(2)    # [pages, kv heads, 1, 2, d]
            q = s["q"][start + j].double().reshape(1, kvh, -1, 1, d)
            score = (q * b).amax(3).sum((2, 3)).transpose(0, 1)                          # [kv heads, pages]
            score = torch.nan_to_num(score, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
            number = torch.arange(mine + 1, device=DEVICE)
            always = (number < FIRST) | (number > mine - LAST)
            # a page's place: those always read ahead of all others, then how many score more, or as much and come before it
            before = (score.unsqueeze(1) > score.unsqueeze(2)) | ((score.unsqueeze(1) == score.unsqueeze(2)) & (number.view(1, -1) < number.view(-1, 1)))
            rest = ~always
            place = torch.where(always, -1, int(always.sum()) + (before & rest).sum(-1))
            for h in range(kvh):
                got = number[place[h] < top]
                out[start + j, h, :got.numel()] = got.to(torch.int32)
    return out
