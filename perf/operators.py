"""Cases of the paged key/value cache's operators: the append with its rotation, the attention
of new tokens over the cache, and the attention over the positions that a top-k selected.

A case is a dict of plain values.  ``op`` names the operator; ``batch`` sequences bring at most
``new`` tokens each and hold at most ``ctx`` positions with them (``ragged``: each sequence has
its own numbers); ``hq`` query heads share ``hkv`` key/value heads of ``d`` features; the
cache's pages hold ``page`` positions.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
THETA = 10000.0

# The sizes that draw() spreads over; the listed cases lie in them.
HEADS = ((32, 8), (16, 16), (16, 2), (8, 1), (12, 4), (64, 8), (20, 4))


def listed():
    base = {"dtype": "bf16", "d": 128, "hq": 32, "hkv": 8, "page": 64, "ragged": False}

    def case(name, op, **kw):
        return {"name": name, "op": op, **base, **kw}

    return [
        # one user's next token: nothing but latency
        case("append_b1", "append", batch=1, new=1, ctx=4096, rope=64, pairs=False),
        # the decode step of a batch of 64 sequences, every head with keys of its own
        case("append_b64", "append", batch=64, new=1, ctx=1024, hq=16, hkv=16, rope=64, pairs=False),
        # prompts of several users in chunks of odd lengths, rotation of neighbouring pairs
        case("append_chunks", "append", batch=8, new=2048, ctx=2500, ragged=True, dtype="f16",
             page=16, rope=128, pairs=True),
        # one user's next token after a long prompt: one row of work for the whole GPU
        case("attend_b1_32k", "attend", batch=1, new=1, ctx=32768, window=0, lse=False),
        # a serving batch with a long and a short tail
        case("attend_b32_ragged", "attend", batch=32, new=1, ctx=16384, ragged=True, page=16,
             window=0, lse=False),
        # a few drafted tokens per sequence checked at once
        case("attend_b16_draft4", "attend", batch=16, new=4, ctx=8192, window=0, lse=True),
        # one chunk of a prompt
        case("attend_chunk512_8k", "attend", batch=1, new=512, ctx=8192, window=0, lse=False),
        # a large chunk late in a long prompt: the largest one
        case("attend_chunk4k_16k", "attend", batch=1, new=4096, ctx=16384, window=0, lse=False),
        # several users' chunks, narrow heads in groups of three, a sliding window
        case("attend_window_ragged", "attend", batch=8, new=700, ctx=6000, ragged=True, dtype="f16",
             hq=12, hkv=4, d=64, page=32, window=1024, lse=True),
        # one sequence's decode step over the 2048 positions its top-k chose
        case("select_b1_32k", "select", batch=1, new=1, ctx=32768, topk=2048),
        # the same for 64 sequences at 32768 positions
        case("select_b64_32k", "select", batch=64, new=1, ctx=32768, topk=2048),
        # chunks of a prompt: a selection for every token, short ones padded with -1
        case("select_chunks", "select", batch=3, new=401, ctx=3500, ragged=True, dtype="f16",
             hq=16, hkv=2, d=64, page=16, topk=512),
    ]


def lengths(case):
    """(new tokens, positions with them) of every sequence; they depend on the case alone."""
    new, ctx = case["new"], case["ctx"]
    if not case["ragged"]:
        return [new] * case["batch"], [max(new, ctx)] * case["batch"]
    ns, ls = [], []
    for i in range(case["batch"]):
        u, v = ((i + 1) * 0.6180339887) % 1.0, ((i + 1) * 0.7548776662) % 1.0
        n = 1 if new == 1 else int(new * u)
        ns.append(n)
        ls.append(max(n, int(ctx * v), 1))
    return ns, ls


def visible(case):
    """Number of (token, key) pairs that attend, and of keys that any token attends to."""
    pairs = keys = 0
    for n, length in zip(*lengths(case)):
        w = case.get("window") or length
        first = length - n
        if n:
            keys += length - max(0, first + 1 - w)
            full = max(0, min(n, w - first))  # tokens whose window starts before position 0
            pairs += full * first + full * (full + 1) // 2 + (n - full) * w
    return pairs, keys


def work(case):
    ns, ls = lengths(case)
    t, e = sum(ns), 2
    row = case["hkv"] * case["d"] * e
    if case["op"] == "append":
        moved = t * (case["hq"] * case["d"] * e + 2 * row)
        return {"bytes": 2 * moved, "flops": 3 * t * (case["hq"] + case["hkv"]) * case["rope"]}
    io = 2 * t * case["hq"] * case["d"] * e
    if case["op"] == "attend":
        pairs, keys = visible(case)
        io += 4 * t * case["hq"] if case["lse"] else 0
    else:
        pairs = keys = 0
        for n, length in zip(ns, ls):
            got = sum(min(case["topk"], length - n + 1 + i) for i in range(n))
            pairs += got
            keys += min(got, length if n else 0)
        io += 4 * t * case["topk"]
    return {"bytes": io + 2 * keys * row, "flops": 4 * pairs * case["hq"] * case["d"]}


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = max(b, w["bytes"]), max(f, w["flops"])
    while True:
        op = rng.choice(("append", "attend", "attend", "select"))
        hq, hkv = rng.choice(HEADS)
        case = {"op": op, "dtype": rng.choice(("bf16", "f16")), "d": rng.choice((64, 128)),
                "hq": hq, "hkv": hkv, "page": rng.choice((16, 32, 64, 128)),
                "ragged": rng.random() < 0.6}
        one = rng.random() < 0.4
        case["batch"] = log(1, 64)
        case["new"] = 1 if one else log(2, 4096)
        case["ctx"] = max(case["new"], log(16, 32768))
        if op == "append":
            case.update(rope=rng.choice((32, 64)) if case["d"] == 64 else rng.choice((64, 128)),
                        pairs=rng.random() < 0.5)
        elif op == "attend":
            case.update(window=0 if rng.random() < 0.7 else log(16, 4096), lse=rng.random() < 0.5)
        else:
            case["topk"] = log(16, 2048)
        ns, ls = lengths(case)
        if sum(ns) == 0:
            continue
        w = work(case)
        # the plain forms hold a value per (padded token, padded position) of every head
        padded = case["batch"] * max(ns) * max(ls) * hq
        gathered = sum(ns) * case.get("topk", 0) * hkv * case["d"]
        cached = sum(ls) * hkv * case["d"]
        if (w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and cached <= 1 << 31
                and (op != "attend" or padded <= 1 << 31) and gathered <= 1 << 30
                and (op != "select" or sum(ns) * max(ls) <= 1 << 24)):
            return case


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    ns, ls = lengths(case)
    t, b, p = sum(ns), case["batch"], case["page"]
    per = [-(-length // p) for length in ls]
    total, width = sum(per) + 3, max(per)
    # pages as a running server leaves them: in no order
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    starts = [0]
    for n in ns:
        starts.append(starts[-1] + n)
    s = {"case": case, "table": table, "max_new": max(ns), "max_len": max(ls),
         "starts": torch.tensor(starts, dtype=torch.int32, device=dev),
         "lengths": torch.tensor(ls, dtype=torch.int32, device=dev),
         "keys": normal(total, p, case["hkv"], case["d"]),
         "values": normal(total, p, case["hkv"], case["d"]),
         "q": normal(t, case["hq"], case["d"])}
    if case["op"] == "append":
        s["k"], s["v"] = normal(t, case["hkv"], case["d"]), normal(t, case["hkv"], case["d"])
        half = case["rope"] // 2
        s["freq"] = THETA ** (-torch.arange(half, device=dev, dtype=torch.float32) / half)
    if case["op"] == "select":
        # what a top-k without an order returns: ascending positions, -1 where there are fewer
        seq, pos = _tokens(s)
        noise = torch.rand(t, s["max_len"], generator=g, device=dev)
        noise.masked_fill_(torch.arange(s["max_len"], device=dev) > pos[:, None], -1.0)
        k = min(case["topk"], s["max_len"])
        top = noise.topk(k, dim=1)
        idx = torch.where(top.values < 0, s["max_len"], top.indices).sort(dim=1).values
        idx = torch.where(idx == s["max_len"], -1, idx).to(torch.int32)
        s["indices"] = torch.nn.functional.pad(idx, (0, case["topk"] - k), value=-1)
    if own:
        from dsa_b200 import paged

        s["cache"] = paged.PagedKV(s["keys"], s["values"])
        s["batch"] = paged.PagedBatch(table, s["starts"], s["lengths"], max_new=s["max_new"])
        if case["op"] == "append":
            s["appender"] = paged.PagedAppender(s["cache"], rope_dim=case["rope"],
                                                inv_freq=s["freq"], interleaved=case["pairs"])
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        from dsa_b200 import paged

        if op == "append":
            q = s["appender"].append(s["batch"], s["k"], s["v"], s["q"])
            return {"q": q, "keys": s["keys"], "values": s["values"]}
        if op == "attend":
            window = s["case"]["window"] or None
            if s["case"]["lse"]:
                out, lse = paged.paged_attention(s["q"], s["cache"], s["batch"], window=window,
                                                 return_lse=True)
                return {"out": out, "lse": lse}
            return {"out": paged.paged_attention(s["q"], s["cache"], s["batch"], window=window)}
        return {"out": paged.selected_attention(s["q"], s["cache"], s["batch"], s["indices"])}
    return {"append": _append, "attend": _attend, "select": _select}[op](s)


# ------------------------------------------------------------------ plain forms, float32

def _tokens(s):
    """Every token's sequence and position."""
    t = torch.arange(s["q"].shape[0], device=s["q"].device)
    starts = s["starts"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    new = starts[1:] - starts[:-1]
    return seq, s["lengths"].long()[seq] - new[seq] + t - starts[seq]


def _rotate(x, pos, freq, pairs):
    angle = pos.float()[:, None] * freq
    cos, sin = angle.cos()[:, None, :], angle.sin()[:, None, :]
    half = freq.shape[0]
    x = x.float()
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if pairs else (rot[..., :half], rot[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack((a, b), -1).flatten(-2) if pairs else torch.cat((a, b), -1)
    return torch.cat((rot, rest), -1)


def _append(s):
    seq, pos = _tokens(s)
    dtype, page, pairs = s["q"].dtype, s["case"]["page"], s["case"]["pairs"]
    at = s["table"].long()[seq, pos // page]
    s["keys"][at, pos % page] = _rotate(s["k"], pos, s["freq"], pairs).to(dtype)
    s["values"][at, pos % page] = s["v"]
    return {"q": _rotate(s["q"], pos, s["freq"], pairs).to(dtype), "keys": s["keys"],
            "values": s["values"]}


def _attend(s):
    case, q, dev = s["case"], s["q"], s["q"].device
    hkv, d, page, group = case["hkv"], case["d"], case["page"], case["hq"] // case["hkv"]
    b, length, new = case["batch"], s["max_len"], s["max_new"]
    table = s["table"].long()
    k = s["keys"][table].reshape(b, -1, hkv, d)[:, :length].float()
    v = s["values"][table].reshape(b, -1, hkv, d)[:, :length].float()
    starts = s["starts"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(new, device=dev)
    row = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)             # [b, new]
    there = i < count[:, None]
    pos = s["lengths"].long()[:, None] - count[:, None] + i
    j = torch.arange(length, device=dev)
    sees = (j <= pos[..., None]) & there[..., None]                     # [b, new, length]
    if case["window"]:
        sees &= j > pos[..., None] - case["window"]
    sees = sees[:, None, None]
    qq = q[row].float().reshape(b, new, hkv, group, d).permute(0, 2, 3, 1, 4)
    sc = (qq.reshape(b, hkv, group * new, d) @ k.permute(0, 2, 3, 1)).view(b, hkv, group, new, length)
    sc.mul_(d ** -0.5).masked_fill_(~sees, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    w = sc.sub_(m).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(b, hkv, group * new, length) @ v.permute(0, 2, 1, 3)).view(b, hkv, group, new, d)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (total.log() + m).squeeze(-1)
    out = torch.zeros(q.shape, dtype=q.dtype, device=dev)
    out[row[there]] = o.permute(0, 3, 1, 2, 4).reshape(b, new, -1, d)[there].to(q.dtype)
    if not case["lse"]:
        return {"out": out}
    all_lse = torch.zeros(q.shape[:2], device=dev)
    all_lse[row[there]] = lse.permute(0, 3, 1, 2).reshape(b, new, -1)[there]
    return {"out": out, "lse": all_lse}


def _select(s):
    case, q = s["case"], s["q"]
    hkv, d, page, group = case["hkv"], case["d"], case["page"], case["hq"] // case["hkv"]
    seq, _ = _tokens(s)
    idx = s["indices"].long()
    there = idx >= 0
    idx = idx.clamp(min=0)
    at = s["table"].long()[seq[:, None], idx // page]
    k = s["keys"][at, idx % page].float().transpose(1, 2)               # [t, hkv, topk, d]
    v = s["values"][at, idx % page].float().transpose(1, 2)
    sc = q.float().view(-1, hkv, group, d) @ k.transpose(2, 3) * d ** -0.5
    sc = sc.masked_fill(~there[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    w = (sc - torch.where(m == -math.inf, 0.0, m)).exp()
    total = w.sum(-1, keepdim=True)
    o = torch.where(total > 0, w @ v / total, 0.0)
    return {"out": o.reshape(q.shape).to(q.dtype)}


# ------------------------------------------------------------------ the definition, float64

def exact(case, seed):
    s = prepare(case, seed)
    ns, ls = lengths(case)
    page, group, d = case["page"], case["hq"] // case["hkv"], case["d"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    keys = values = None
    if case["op"] == "append":
        keys, values = s["keys"].double(), s["values"].double()
    start = 0
    for i, (n, length) in enumerate(zip(ns, ls)):
        rows = slice(start, start + n)
        start += n
        if not n:
            continue
        pages = s["table"][i, :-(-length // page)].long()
        where = torch.arange(length - n, length, device=q.device)
        if case["op"] == "append":
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=q.device),
                               torch.outer(where.double(), s["freq"].double()))
            slot = pages[where // page], where % page
            out[rows] = _turned(q[rows], turn, case["pairs"])
            keys[slot] = _turned(s["k"][rows].double(), turn, case["pairs"])
            values[slot] = s["v"][rows].double()
            continue
        kept = s["keys"][pages].flatten(0, 1)[:length]
        vals = s["values"][pages].flatten(0, 1)[:length]
        for h in range(case["hkv"]):
            heads = slice(h * group, h * group + group)
            kh, vh = kept[:, h].double(), vals[:, h].double()
            if case["op"] == "attend":
                far = where[:, None] - torch.arange(length, device=q.device)
                hidden = (far < 0) | (far >= case["window"] if case["window"] else far < 0)
                for head in range(heads.start, heads.stop):
                    z = torch.einsum("nd,ld->nl", q[rows, head], kh).div_(math.sqrt(d))
                    z.masked_fill_(hidden, -math.inf)
                    lse[rows, head] = torch.logsumexp(z, 1)
                    out[rows, head] = torch.softmax(z, 1) @ vh
            else:
                for lo in range(rows.start, rows.stop, 256):
                    part = slice(lo, min(lo + 256, rows.stop))
                    idx = s["indices"][part].long()
                    gone = idx < 0
                    z = torch.einsum("ngd,nld->ngl", q[part, heads], kh[idx.clamp(min=0)])
                    z = z.div_(math.sqrt(d)).masked_fill_(gone[:, None], -math.inf)
                    out[part, heads] = torch.softmax(z, 2) @ vh[idx.clamp(min=0)]
    if case["op"] == "append":
        return {"q": out, "keys": keys, "values": values}
    return {"out": out, "lse": lse} if case.get("lse") else {"out": out}


def _turned(x, turn, pairs):
    """x's leading features as complex numbers, multiplied by the unit numbers ``turn``."""
    half = turn.shape[1]
    lead = x[..., :2 * half]
    lead = lead.unflatten(-1, (half, 2)) if pairs else lead.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(lead.contiguous()) * turn[:, None])
    z = z.flatten(-2) if pairs else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., 2 * half:]), -1)
