"""The work that is timed: what a serving program does around its quantized projections.

A case is one pass through an operator of the public entry points on inputs
made from a seed.  `listed()` holds the fixed cases, `draw(rng)` more of the
same ranges:

- attend: one new token per sequence attends to the sequence's pages of the
  key-value cache (any lengths, grouped heads, a window, sinks, a soft cap).
- grow: the pages for new tokens are reserved, and one layer's keys and values
  of the tokens are written to them: a decode step, or a chunk of prompts.
- fork: sequences split into several that share their full pages; the last,
  part-full page is copied in every pool (one per layer, keys and values).
- compact: sequences leave, their pages are freed, and the pages that are left
  move to the front of every pool.
- norm: the residual update and the norms around it.
- logprobs: log probabilities of given tokens, entropy and top alternatives of
  a step's or a prompt's logits.

With `own` false `run` computes the same in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases -------------------------------------------------------------------


def _attend(name, B, Hq, Hkv, D, length, page, dtype="bf16", ragged=False, window=0, sinks=False, softcap=0.0):
    return {"name": name, "kind": "attend", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "length": length, "page": page,
            "dtype": dtype, "ragged": ragged, "window": window, "sinks": sinks, "softcap": softcap}


def listed():
    return [
        # a chat's first answer: one sequence of 200 tokens, the smallest call, latency
        _attend("attend_1_200", 1, 32, 8, 128, 200, 16),
        # a serving batch of 32 conversations of all lengths up to 8000 tokens
        _attend("attend_32_ragged", 32, 32, 4, 128, 8000, 16, ragged=True),
        # 64 sequences in a layer with a window of 128 tokens and a sink per head
        _attend("attend_64_window", 64, 64, 8, 64, 4000, 32, ragged=True, window=128, sinks=True),
        # four documents of 131072 tokens: the largest read
        _attend("attend_4_131072", 4, 32, 8, 128, 131072, 64, dtype="f16"),
        # a decode step of 64 sequences: one token each
        {"name": "grow_step_64", "kind": "grow", "R": 64, "new": 1, "length": 3000, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "bf16"},
        # a chunk of three prompts, 4098 tokens together
        {"name": "grow_prompts_4098", "kind": "grow", "R": 3, "new": 1366, "length": 700, "Hkv": 8, "D": 128,
         "page": 16, "dtype": "f16"},
        # four prompts answered eight times each, over the 72 pools of 36 layers
        {"name": "fork_4x8", "kind": "fork", "R": 4, "ways": 8, "length": 1500, "Hkv": 8, "D": 128, "page": 16,
         "pools": 72, "dtype": "bf16"},
        # 24 of 64 sequences leave, the rest moves to the front of 16 pools
        {"name": "compact_24_of_64", "kind": "compact", "R": 64, "leave": 24, "length": 700, "Hkv": 8, "D": 128,
         "page": 16, "pools": 16, "dtype": "bf16"},
        # one token's residual update and the norm of the next block: latency
        {"name": "norm_1_4096", "kind": "norm", "T": 1, "H": 4096, "dtype": "bf16", "post": False, "gate": "none",
         "scale": 1.0, "offset": 0.0},
        # a prompt chunk of 2047 tokens, norms on both sides of the block, gated per token
        {"name": "norm_2047_2880", "kind": "norm", "T": 2047, "H": 2880, "dtype": "bf16", "post": True,
         "gate": "token", "scale": 0.22, "offset": 1.0},
        # the token just sampled, its entropy and 20 alternatives
        {"name": "logprobs_1_151936", "kind": "logprobs", "T": 1, "V": 151936, "dtype": "bf16", "tokens": 1, "k": 20,
         "scale": 1.0},
        # scoring a prompt chunk: 300 positions in 32 bits, 5 alternatives each
        {"name": "logprobs_300_151936", "kind": "logprobs", "T": 300, "V": 151936, "dtype": "f32", "tokens": 1,
         "k": 5, "scale": 0.7},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "grow", "fork", "compact", "norm", "norm", "logprobs", "logprobs"))
    if kind == "attend":
        Hkv = rng.choice((1, 2, 4, 8, 16))
        Hq = Hkv * rng.choice((1, 2, 4, 5, 8, 16))
        D = rng.choice((64, 80, 96, 128, 128, 192, 256))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        B = _log_int(rng, 1, 200)
        most = (4 * 131072 * 8 * 128 * 2) // (B * Hkv * D * _SIZES[dtype])
        length = min(_log_int(rng, 1, 140000), max(1, most // 2))
        return {"kind": "attend", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "length": length,
                "page": rng.choice((8, 16, 16, 32, 64, 24)), "dtype": dtype, "ragged": rng.random() < 0.6,
                "window": rng.choice((0, 0, 0, 128, 1000)), "sinks": rng.random() < 0.25,
                "softcap": rng.choice((0.0, 0.0, 0.0, 30.0))}
    if kind in ("grow", "fork", "compact"):
        Hkv, D = rng.choice((1, 2, 4, 8)), rng.choice((64, 96, 128, 256))
        page, dtype = rng.choice((8, 16, 16, 32)), rng.choice(("bf16", "f16", "f32"))
        base = {"kind": kind, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype}
        if kind == "grow":
            R = _log_int(rng, 1, 128)
            return {**base, "R": R, "new": rng.choice((1, _log_int(rng, 1, max(1, 4000 // R)))),
                    "length": _log_int(rng, 10, 3000)}
        pools = rng.choice((2, 8, 16, 48))
        # at most the listed sizes: bytes of all pools
        room = (1 << 30) // (pools * Hkv * D * _SIZES[dtype])
        if kind == "fork":
            R = _log_int(rng, 1, 8)
            ways = rng.choice((1, 2, 4, 8))
            return {**base, "R": R, "ways": ways, "pools": pools,
                    "length": min(_log_int(rng, 10, 3000), max(10, room // (2 * R) - page * ways))}
        R = _log_int(rng, 2, 64)
        return {**base, "R": R, "leave": max(1, int(R * rng.uniform(0.1, 0.9))), "pools": pools,
                "length": min(_log_int(rng, 10, 2000), max(10, room // R))}
    if kind == "norm":
        H = rng.choice((64, 512, 1152, 2048, 2880, 4096, 5120, 8192, _log_int(rng, 100, 12000)))
        T = min(_log_int(rng, 1, 4096), max(1, 2047 * 2880 * 2 // H))
        return {"kind": "norm", "T": T, "H": H, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
                "post": rng.random() < 0.5, "gate": rng.choice(("none", "none", "channel", "token", "row")),
                "scale": rng.choice((1.0, 0.22, 1.4)), "offset": rng.choice((0.0, 0.0, 1.0))}
    V = rng.choice((32000, 50257, 128256, 151936, 201088, 262144, _log_int(rng, 50, 200000)))
    T = min(_log_int(rng, 1, 2000), max(1, 300 * 151936 // V))
    return {"kind": "logprobs", "T": T, "V": V, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
            "tokens": rng.choice((1, 1, 1, 4)), "k": min(V, rng.choice((0, 1, 5, 20, 20, 64))),
            "scale": rng.choice((1.0, 1.0, 0.7, 1.6))}


def _lengths(n, length, ragged):
    """n sequence lengths up to `length`: equal, or spread over the whole range."""
    if not ragged:
        return [length] * n
    return [max(1, round(length * (((i + 1) * 0.6180339887498949) % 1.0) ** 2)) for i in range(n)]


def _cdiv(a, b):
    return -(-a // b)


# ---- inputs --------------------------------------------------------------------


def _placed(lengths, page, pages, gen):
    """A table [len(lengths), widest] of pages dealt out in random order (-1: none), and the order."""
    per = [_cdiv(n, page) for n in lengths]
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lengths), max(1, max(per))), -1, dtype=torch.int64)
    at = torch.cumsum(torch.tensor([0] + per), 0)
    j = torch.arange(table.shape[1])
    live = j[None] < torch.tensor(per)[:, None]
    table[live] = order[(at[:-1, None] + j[None])[live]]
    return table, order


def _values(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    dt = _DTYPES[case["dtype"]]
    if kind == "attend":
        B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
        lengths = _lengths(B, case["length"], case["ragged"])
        pages = sum(_cdiv(n, page) for n in lengths) + 5
        table, _ = _placed(lengths, page, pages, host)
        s["table"] = table.clamp(min=0).int().cuda()
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
        s["q"] = _values((B, case["Hq"], D), dt, gen)
        s["k"], s["v"] = (_values((pages, Hkv, page, D), dt, gen) for _ in range(2))
        s["sinks"] = torch.randn(case["Hq"], generator=gen, device="cuda") if case["sinks"] else None
        return s
    if kind in ("grow", "fork", "compact"):
        R, page, D, Hkv = case["R"], case["page"], case["D"], case["Hkv"]
        lengths = _lengths(R, case["length"], True)
        rows, new = R, 0
        if kind == "grow":
            # every row by about `new` tokens
            counts = [case["new"] if case["new"] == 1 else max(1, case["new"] + (i % 3 - 1) * (case["new"] // 4))
                      for i in range(R)]
            new = sum(_cdiv(n + c, page) - _cdiv(n, page) for n, c in zip(lengths, counts))
            width = max(_cdiv(n + c, page) for n, c in zip(lengths, counts))
        elif kind == "fork":
            rows = R * (1 + case["ways"])
            new, width = R * case["ways"], max(_cdiv(n, page) for n in lengths)
        else:
            width = max(_cdiv(n, page) for n in lengths)
        used = sum(_cdiv(n, page) for n in lengths)
        pages = used + new + max(4, used // 8)
        small, _ = _placed(lengths, page, pages, host)
        table = torch.full((rows, width), -1, dtype=torch.int64)
        table[:R, :min(width, small.shape[1])] = small[:, :width]
        refs = torch.zeros(pages, dtype=torch.int64)
        refs[small[small >= 0]] = 1
        full = torch.zeros(rows, dtype=torch.int64)
        full[:R] = torch.tensor(lengths)
        # the cache's bookkeeping in one buffer, so that one copy brings it back
        s["book"] = torch.cat([table.reshape(-1), full, refs]).int().cuda()
        s["dims"] = (rows, width, pages)
        pools = case.get("pools", 2)
        s["pools"] = _values((pools, pages, Hkv, page, D), dt, gen)
        s["pool_list"] = list(s["pools"].unbind(0))
        if kind == "grow":
            s["counts"] = torch.tensor(counts, dtype=torch.int32).cuda()
            s["rows"] = torch.cat([torch.full((c,), i) for i, c in enumerate(counts)]).int().cuda()
            s["positions"] = torch.cat([torch.arange(n, n + c) for n, c in zip(lengths, counts)]).int().cuda()
            s["k"], s["v"] = (_values((sum(counts), Hkv, D), dt, gen) for _ in range(2))
        elif kind == "fork":
            s["src"] = torch.arange(R).repeat_interleave(case["ways"]).int().cuda()
            s["dst"] = torch.arange(R, rows).int().cuda()
        else:
            s["leave"] = torch.randperm(R, generator=host)[:case["leave"]].int().cuda()
        return s
    if kind == "norm":
        T, H = case["T"], case["H"]
        s["x"] = _values((T, H), dt, gen)
        s["y"] = _values((T, H), dt, gen)
        s["pre"] = 1.0 - case["offset"] + 0.1 * torch.randn(H, generator=gen, device="cuda")
        s["pre"] = s["pre"].to(dt)
        s["post"] = (1.0 - case["offset"] + 0.1 * torch.randn(H, generator=gen, device="cuda")).to(dt) if case["post"] else None
        shape = {"none": None, "channel": (H,), "token": (T, H), "row": (T, 1)}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(torch.randn(shape, generator=gen, device="cuda")).to(dt)
        return s
    T, V = case["T"], case["V"]
    s["logits"] = (3.0 * torch.randn((T, V), generator=gen, device="cuda")).to(dt)
    s["tokens"] = torch.randint(0, V, (T, case["tokens"]), generator=gen, device="cuda", dtype=torch.int32)
    return s


# ---- one pass --------------------------------------------------------------------


def _book(s):
    rows, width, pages = s["dims"]
    book = s["book"].clone()
    return (book[:rows * width].view(rows, width), book[rows * width:rows * width + rows],
            book[rows * width + rows:])


def _run_own(s):
    import mlxcel_amd as mq

    c = s["case"]
    kind = c["kind"]
    if kind == "attend":
        return mq.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=c["window"],
                                  softcap=c["softcap"], sinks=s["sinks"])
    if kind == "norm":
        return mq.residual_norm(s["x"], s["y"], post_weight=s["post"], gate=s["gate"], scale=c["scale"],
                                pre_weight=s["pre"], eps=1e-6, weight_offset=c["offset"])
    if kind == "logprobs":
        return mq.token_logprobs(s["logits"], s["tokens"], top_k=c["k"], scale=c["scale"])
    table, lengths, refs = _book(s)
    if kind == "grow":
        granted = mq.cache_reserve(table, lengths, refs, s["counts"], c["page"])
        mq.cache_append(s["k"], s["v"], s["pool_list"][0], s["pool_list"][1], table, s["positions"], s["rows"])
        return granted, table, lengths, refs, s["pools"]
    if kind == "fork":
        granted = mq.cache_fork(s["pool_list"], table, lengths, refs, s["src"], s["dst"])
        return granted, table, lengths, refs, s["pools"]
    mq.cache_free(table, lengths, refs, s["leave"], c["page"])
    live = mq.cache_compact(s["pool_list"], table, lengths, refs)
    return live, table, lengths, refs, s["pools"]


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, D, page = c["B"], c["Hq"], c["Hkv"], c["D"], c["page"]
    table = s["table"].long()
    n = table.shape[1] * page

    def rows(pool):
        return pool[table].permute(0, 2, 1, 3, 4).reshape(B * Hkv, n, D).float()

    q = s["q"].float().reshape(B * Hkv, Hq // Hkv, D)
    x = torch.matmul(q, rows(s["k"]).transpose(1, 2)) * (1.0 / math.sqrt(D))
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    at = torch.arange(n, device=q.device)
    keep = at[None] < s["lengths"][:, None]
    if c["window"]:
        keep = keep & (at[None] >= s["lengths"][:, None] - c["window"])
    keep = keep[:, None, None].expand(B, Hkv, 1, n).reshape(B * Hkv, 1, n)
    x = torch.where(keep, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].reshape(1, Hkv, Hq // Hkv, 1).expand(B, -1, -1, -1).reshape(B * Hkv, -1, 1)
        m = torch.maximum(m, sink)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - m)
    return (torch.matmul(p, rows(s["v"])) / total).reshape(B, Hq, D).to(s["q"].dtype)


def _free_first(refs):
    """The free pages in ascending order, in front of the others; how many there are; each page's rank."""
    free = refs == 0
    return torch.argsort((~free).int(), stable=True), free.sum(), torch.cumsum(free, 0) - 1, free


def _plain_reserve(table, lengths, refs, counts, page):
    width = table.shape[1]
    had, want = (lengths + page - 1) // page, (lengths + counts + page - 1) // page
    fits = want <= width
    need = torch.where(fits, want - had, 0)
    last = torch.cumsum(need, 0)
    order, n_free, rank, free = _free_first(refs)
    granted = fits & ((need == 0) | (last <= n_free))
    need = torch.where(granted, need, 0)
    first = torch.cumsum(need, 0) - need
    j = torch.arange(width, device=table.device)[None] - had[:, None]
    mine = (j >= 0) & (j < need[:, None])
    pages = order[(first[:, None] + j).clamp(0, refs.numel() - 1)]
    table.copy_(torch.where(mine, pages, table))
    refs.copy_(torch.where(free & (rank < need.sum()), 1, refs))
    lengths.copy_(torch.where(granted, lengths + counts, lengths))
    return granted.int()


def _plain_fork(pools, table, lengths, refs, src, dst, page):
    src, dst = src.long(), dst.long()
    n = lengths[src]
    full, part = n // page, (n % page != 0).int()
    order, n_free, rank, free = _free_first(refs)
    last = torch.cumsum(part, 0)
    granted = (lengths[dst] == 0) & ((part == 0) | (last <= n_free))
    fresh = order[(last - 1).clamp(0, refs.numel() - 1)]
    j = torch.arange(table.shape[1], device=table.device)[None]
    shared = granted[:, None] & (j < full[:, None])
    mine = granted[:, None] & (j == full[:, None]) & (part[:, None] > 0)
    theirs = table[src]
    table[dst] = torch.where(shared, theirs, torch.where(mine, fresh[:, None], table[dst])).int()
    refs.index_add_(0, theirs.clamp(min=0).reshape(-1), shared.reshape(-1).int())
    copied = torch.nonzero(granted & (part > 0))[:, 0]
    old = theirs.gather(1, full.clamp(max=table.shape[1] - 1)[:, None].long())[:, 0]
    pools[:, fresh[copied]] = pools[:, old[copied].long()]
    refs[fresh[copied]] = 1
    lengths[dst] = torch.where(granted, n, lengths[dst])
    return granted.int()


def _plain_free(table, lengths, refs, rows, page):
    rows = rows.long()
    j = torch.arange(table.shape[1], device=table.device)[None]
    held = j < ((lengths[rows] + page - 1) // page)[:, None]
    refs.index_add_(0, table[rows].clamp(min=0).reshape(-1), -held.reshape(-1).int())
    lengths[rows] = 0


def _plain_compact(pools, table, lengths, refs, page):
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    holes, movers = torch.nonzero(~live & (at < n))[:, 0], torch.nonzero(live & (at >= n))[:, 0]
    to = at.int()
    to[movers] = holes.int()
    j = torch.arange(table.shape[1], device=table.device)[None]
    held = j < ((lengths + page - 1) // page)[:, None]
    table.copy_(torch.where(held, to[table.clamp(min=0)], table))
    pools[:, holes] = pools[:, movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    return n.int().reshape(1)


def _plain_norm(s):
    c = s["case"]
    y = s["y"].float()
    if s["post"] is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * (s["post"].float() + c["offset"])
    if s["gate"] is not None:
        y = y * s["gate"].float()
    h = s["x"].float() + c["scale"] * y
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * (s["pre"].float() + c["offset"])
    return h.to(s["x"].dtype), n.to(s["x"].dtype)


def _plain_logprobs(s):
    c, V = s["case"], s["case"]["V"]
    x = s["logits"].float()
    z = x * c["scale"]
    z = z - z.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(z).sum(-1, keepdim=True))
    lp = z - lse
    entropy = -(torch.exp(lp) * lp).sum(-1)
    given = lp.gather(1, s["tokens"].long())
    if not c["k"]:
        return given, entropy, None, None
    # one whole number per value: larger values first, among equals the lowest index
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + (V - 1 - torch.arange(V, device=x.device))
    ids = torch.topk(order, c["k"], dim=-1)[1]
    return given, entropy, lp.gather(1, ids), ids.int()


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    kind = c["kind"]
    if kind == "attend":
        return _plain_attend(s)
    if kind == "norm":
        return _plain_norm(s)
    if kind == "logprobs":
        return _plain_logprobs(s)
    table, lengths, refs = _book(s)
    if kind == "grow":
        granted = _plain_reserve(table, lengths, refs, s["counts"], c["page"])
        pos = s["positions"].long()
        page = table[s["rows"].long(), pos // c["page"]].long()
        s["pools"][0][page, :, pos % c["page"]] = s["k"]
        s["pools"][1][page, :, pos % c["page"]] = s["v"]
        return granted, table, lengths, refs, s["pools"]
    if kind == "fork":
        granted = _plain_fork(s["pools"], table, lengths, refs, s["src"], s["dst"], c["page"])
        return granted, table, lengths, refs, s["pools"]
    _plain_free(table, lengths, refs, s["leave"], c["page"])
    live = _plain_compact(s["pools"], table, lengths, refs, c["page"])
    return live, table, lengths, refs, s["pools"]


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    """Bytes: each input read once, each output written once; operations of the products and sums."""
    kind, e = case["kind"], _SIZES[case["dtype"]]
    if kind == "attend":
        lengths = _lengths(case["B"], case["length"], case["ragged"])
        seen = sum(min(n, case["window"] or n) for n in lengths)
        token = 2 * case["Hkv"] * case["D"] * e
        return {"bytes": seen * token + 2 * case["B"] * case["Hq"] * case["D"] * e + 4 * seen / case["page"],
                "flops": 4 * seen * case["Hq"] * case["D"]}
    if kind in ("grow", "fork", "compact"):
        page, R = case["page"], case["R"]
        lengths = _lengths(R, case["length"], True)
        page_bytes = case["Hkv"] * case["D"] * page * e
        used = sum(_cdiv(n, page) for n in lengths)
        if kind == "grow":
            tokens = R * case["new"]
            return {"bytes": 4 * tokens * case["Hkv"] * case["D"] * e + 8 * tokens + 16 * R, "flops": 0}
        if kind == "fork":
            copied = case["ways"] * sum(n % page != 0 for n in lengths)
            return {"bytes": 2 * copied * page_bytes * case["pools"] + 16 * case["ways"] * used, "flops": 0}
        pages = used + max(4, used // 8)
        live = used * (R - case["leave"]) / R
        moved = live * (1 - live / pages)  # expected: pages lie in random order
        return {"bytes": 2 * moved * page_bytes * case["pools"] + 8 * pages + 8 * used, "flops": 0}
    if kind == "norm":
        T, H = case["T"], case["H"]
        gate = {"none": 0, "channel": H, "token": T * H, "row": T}[case["gate"]]
        return {"bytes": (4 * T * H + gate + (2 if case["post"] else 1) * H) * e, "flops": 10 * T * H}
    T, V = case["T"], case["V"]
    return {"bytes": T * V * e + T * (8 * case["tokens"] + 4 + 8 * case["k"]), "flops": 5 * T * V}


# ---- 64-bit results ------------------------------------------------------------------


def _exact_attend(s):
    c = s["case"]
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - c["window"]) if c["window"] else 0
        pos = torch.arange(first, n, device="cuda")
        page = s["table"][b].long()[pos // c["page"]]
        for h in range(c["Hkv"]):
            k, v = (s[p][page, h, pos % c["page"]].double() for p in "kv")
            x = s["q"][b, h * G:(h + 1) * G].double() @ k.t() / math.sqrt(c["D"])
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h * G:(h + 1) * G, None].double()], 1)
            p = torch.softmax(x, 1)[:, :n - first]
            out[b, h * G:(h + 1) * G] = p @ v
    return out


def _exact_pages(s):
    """The bookkeeping step by step on the host, with the copies that it names."""
    c = s["case"]
    page, kind = c["page"], c["kind"]
    rows, width, pages = s["dims"]
    book = s["book"].cpu().numpy().astype(np.int64)
    table, lengths = book[:rows * width].reshape(rows, width).copy(), book[rows * width:rows * width + rows].copy()
    refs = book[rows * width + rows:].copy()
    pools = s["pools"].double()
    if kind == "grow":
        given = []
        for r, count in enumerate(s["counts"].tolist()):
            a, b = _cdiv(int(lengths[r]), page), _cdiv(int(lengths[r]) + count, page)
            free = np.flatnonzero(refs == 0)[:b - a]
            ok = b <= width and len(free) == b - a
            if ok:
                table[r, a:b] = free
                refs[free] = 1
                lengths[r] += count
            given.append(int(ok))
        for i, src in enumerate((s["k"], s["v"])):
            for r in range(rows):
                mine = torch.nonzero(s["rows"] == r)[:, 0]
                pos = s["positions"][mine].long()
                at = torch.from_numpy(table[r]).cuda()[pos // page]
                pools[i][at, :, pos % page] = src[mine].double()
        first = np.array(given)
    elif kind == "fork":
        given, start = [], s["pools"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            full, part = divmod(int(lengths[a]), page)
            free = np.flatnonzero(refs == 0)[:1]
            ok = lengths[b] == 0 and (part == 0 or len(free) == 1)
            if ok:
                table[b, :full] = table[a, :full]
                refs[table[a, :full]] += 1
                if part:
                    table[b, full] = free[0]
                    refs[free[0]] = 1
                    pools[:, free[0]] = start[:, table[a, full]]
                lengths[b] = lengths[a]
            given.append(int(ok))
        first = np.array(given)
    else:
        for r in s["leave"].tolist():
            refs[table[r, :_cdiv(int(lengths[r]), page)]] -= 1
            lengths[r] = 0
        n = int((refs > 0).sum())
        to = {}
        for hole, mover in zip(np.flatnonzero(refs[:n] == 0), n + np.flatnonzero(refs[n:] > 0)):
            to[int(mover)] = int(hole)
            refs[hole], refs[mover] = refs[mover], 0
        for r in range(rows):
            for j in range(_cdiv(int(lengths[r]), page)):
                table[r, j] = to.get(int(table[r, j]), table[r, j])
        if to:
            pools[:, list(to.values())] = pools[:, list(to)]
        first = np.array([n])
    return first, table, lengths, refs, pools


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend":
        return _exact_attend(s)
    if kind in ("grow", "fork", "compact"):
        return _exact_pages(s)
    if kind == "norm":
        def rms(t, w):
            return t / torch.sqrt(t.pow(2).sum(-1, keepdim=True) / case["H"] + 1e-6) * (w.double() + case["offset"])

        y = s["y"].double()
        y = rms(y, s["post"]) if s["post"] is not None else y
        h = s["x"].double() + case["scale"] * (y if s["gate"] is None else y * s["gate"].double())
        return h, rms(h, s["pre"])
    lp = torch.log_softmax(s["logits"].double() * case["scale"], -1)
    given = torch.stack([lp[torch.arange(case["T"], device="cuda"), t.long()] for t in s["tokens"].unbind(1)], 1)
    entropy = torch.special.entr(torch.exp(lp)).sum(-1)
    if not case["k"]:
        return given, entropy, None, None
    ids = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)[1][:, :case["k"]]
    return given, entropy, lp.gather(1, ids), ids
