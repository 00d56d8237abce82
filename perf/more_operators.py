"""The work that is timed: a prompt's way into the paged cache and a step's way out of the logits.

A case is one pass through an operator of the public entry points on inputs
made from a seed.  `listed()` holds the fixed cases, `draw(rng)` more of the
same ranges:

- rotary: the position rotation of heads (half or interleaved pairs, all of a
  head or its first part, far positions), read from a fused projection's rows.
- append: queries are rotated, keys are rotated on their way into the pages of
  the key-value cache, values are written beside them.
- chunk: several new tokens per sequence attend to the sequence's pages and to
  one another (prompts, parts of prompts, drafted tokens, single tokens among
  them), with grouped heads, a window, sinks, a soft cap.
- adjust: penalties for the tokens of a history, biases of single tokens and a
  grammar's mask on a step's logits.

With `own` false `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases -------------------------------------------------------------------


def _rotary(name, T, H, D, dims, dtype="bf16", interleaved=False, far=0, factor=1.0):
    return {"name": name, "kind": "rotary", "T": T, "H": H, "D": D, "dims": dims, "dtype": dtype,
            "interleaved": interleaved, "far": far, "factor": factor}


def _append(name, R, new, length, Hq, Hkv, D, dims, page, dtype="bf16", interleaved=False, factor=1.0):
    return {"name": name, "kind": "append", "R": R, "new": new, "length": length, "Hq": Hq, "Hkv": Hkv, "D": D,
            "dims": dims, "page": page, "dtype": dtype, "interleaved": interleaved, "factor": factor}


def _chunk(name, B, singles, new, cached, Hq, Hkv, D, page, dtype="bf16", window=0, sinks=False, softcap=0.0):
    return {"name": name, "kind": "chunk", "B": B, "singles": singles, "new": new, "cached": cached, "Hq": Hq,
            "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "softcap": softcap}


def _adjust(name, T, V, history, dtype="bf16", penalties=True, bias=0, mask=False):
    return {"name": name, "kind": "adjust", "T": T, "V": V, "history": history, "dtype": dtype,
            "penalties": penalties, "bias": bias, "mask": mask}


def listed():
    return [
        # one token's query heads: latency
        _rotary("rotary_1", 1, 32, 128, 128),
        # a long document's queries from position 120000 on, the first 64 of 96 elements in interleaved pairs
        _rotary("rotary_8191_part", 8191, 32, 96, 64, dtype="f16", interleaved=True, far=120000, factor=1.2),
        # a decode step of 64 sequences: one token each
        _append("append_step_64", 64, 1, 3000, 32, 8, 128, 128, 16),
        # a chunk of three prompts, 4098 tokens together
        _append("append_prompts_4098", 3, 1366, 700, 32, 8, 128, 128, 16, factor=1.1),
        # a short question into an empty cache: the smallest call, latency
        _chunk("chunk_1_33", 1, 0, 33, 0, 32, 8, 128, 16),
        # five drafted tokens of each of 16 conversations of all lengths up to 8000 tokens
        _chunk("chunk_16x5_ragged", 16, 0, 5, 8000, 32, 4, 128, 16),
        # 61 sequences go on by a token while three prompts are read, about 1000 tokens each
        _chunk("chunk_3_prompts_61_singles", 64, 61, 1000, 3000, 40, 8, 128, 16, dtype="f16"),
        # five prompts in a layer with a window of 128 tokens and a sink per head
        _chunk("chunk_5_window", 5, 0, 1500, 700, 64, 8, 64, 32, window=128, sinks=True),
        # a part of a document of 32768 tokens: the largest products
        _chunk("chunk_2048_of_32768", 1, 0, 2048, 30720, 32, 8, 128, 64),
        # the logits of one answer of 500 tokens: latency
        _adjust("adjust_1_151936", 1, 151936, 500),
        # a batch of 128 long answers under penalties, biases and a grammar
        _adjust("adjust_128_151936", 128, 151936, 4000, bias=300, mask=True),
        # 17 answers of an object's fields: a grammar's mask alone, in 32 bits
        _adjust("adjust_17_128256_mask", 17, 128256, 0, dtype="f32", penalties=False, mask=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "append", "chunk", "chunk", "chunk", "chunk", "adjust", "adjust"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    D = rng.choice((64, 80, 96, 128, 128, 192, 256))
    dims = D if rng.random() < 0.6 else rng.choice((D // 2, D // 4))
    turn = {"interleaved": rng.random() < 0.4, "factor": rng.choice((1.0, 1.0, 1.2))}
    if kind == "rotary":
        H = rng.choice((1, 2, 4, 8, 20, 32, 64))
        T = min(_log_int(rng, 1, 9000), max(1, 8191 * 32 * 96 * 2 // (H * D * _SIZES[dtype])))
        return {"kind": kind, "T": T, "H": H, "D": D, "dims": dims, "dtype": dtype, **turn,
                "far": rng.choice((0, 0, 5000, 120000, 1000000))}
    Hkv = rng.choice((1, 2, 4, 8, 16))
    Hq = Hkv * rng.choice((1, 2, 4, 5, 8))
    page = rng.choice((8, 16, 16, 32, 64, 24))
    if kind == "append":
        R = _log_int(rng, 1, 128)
        most = 4098 * 48 * 128 * 2 // (R * (Hq + 2 * Hkv) * D * _SIZES[dtype])
        return {"kind": kind, "R": R, "new": max(1, min(most, rng.choice((1, _log_int(rng, 1, max(1, 4000 // R)))))),
                "length": _log_int(rng, 10, 3000), "Hq": Hq, "Hkv": Hkv, "D": D, "dims": dims, "page": page,
                "dtype": dtype, **turn}
    if kind == "chunk":
        B = _log_int(rng, 1, 80)
        singles = rng.choice((0, 0, B // 2, B - 1))
        new = _log_int(rng, 1, 3000)
        cached = rng.choice((0, _log_int(rng, 10, 40000)))
        # at most the largest listed case's products, in 32 bits a hundredth, and 256 MiB of cache
        room = (3e9 if dtype == "f32" else 2.6e11) / (Hq * D)
        cached = min(cached, int(2 ** 27 / (B * Hkv * D * _SIZES[dtype])))
        tokens = max(1, min(int(room / (cached + 1)), int(math.sqrt(room))))
        return {"kind": kind, "B": B, "singles": singles, "new": max(1, min(new, tokens // (B - singles))),
                "cached": cached, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype,
                "window": rng.choice((0, 0, 0, 128, 1000)), "sinks": rng.random() < 0.25,
                "softcap": rng.choice((0.0, 0.0, 0.0, 30.0))}
    V = rng.choice((32000, 50257, 128256, 151936, 201088, 262144, _log_int(rng, 50, 200000)))
    T = min(_log_int(rng, 1, 500), max(1, 128 * 151936 * 2 // (V * _SIZES[dtype])))
    penalties = rng.random() < 0.8
    bias = rng.choice((0, 1, 20, 300))
    return {"kind": kind, "T": T, "V": V, "history": _log_int(rng, 1, 4000) if penalties else 0, "dtype": dtype,
            "penalties": penalties, "bias": bias, "mask": rng.random() < 0.5 or not (penalties or bias)}


def _cdiv(a, b):
    return -(-a // b)


def _spread(n, most):
    """n lengths over the whole range up to `most`."""
    return [max(1, round(most * (((i + 1) * 0.6180339887498949) % 1.0) ** 2)) for i in range(n)]


def _news(case):
    """New tokens of each sequence of an append or chunk case, and the tokens it had."""
    if case["kind"] == "append":
        R, new = case["R"], case["new"]
        return [new if new == 1 else max(1, new + (i % 3 - 1) * (new // 4)) for i in range(R)], _spread(R, case["length"])
    B, new = case["B"], case["new"]
    news = [1 if i < case["singles"] else max(1, new + (i % 3 - 1) * (new // 8)) for i in range(B)]
    if B == 1:
        return [new], [case["cached"]]
    return news, _spread(B, case["cached"]) if case["cached"] else [0] * B


def _seen(case):
    """Keys that are read, and (token, key) pairs, of a chunk case."""
    keys = pairs = 0
    for n, had in zip(*_news(case)):
        w = case["window"] or had + n
        keys += min(had + n, w + n - 1)
        # token i sees min(had + i + 1, w) keys
        short = min(n, max(0, w - had))
        pairs += short * had + short * (short + 1) // 2 + (n - short) * w
    return keys, pairs


# ---- inputs --------------------------------------------------------------------


def _values(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _frequencies(dims):
    """Frequencies for long contexts: slow ones are a quarter, as positions are four times those of training."""
    inv = 500000.0 ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    return torch.where(inv < 2 * math.pi / 2048, inv / 4, inv).float().cuda()


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    dt = _DTYPES[case["dtype"]]
    if kind == "rotary":
        # the heads are the first half of a projection's rows
        s["qkv"] = _values((case["T"], 2 * case["H"] * case["D"]), dt, gen)
        s["positions"] = (case["far"] + torch.arange(case["T"])).int().cuda()
        s["inv_freq"] = _frequencies(case["dims"])
        return s
    if kind in ("append", "chunk"):
        Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
        news, had = _news(case)
        lengths = [a + b for a, b in zip(news, had)]
        per = [_cdiv(n, page) for n in lengths]
        pages = sum(per) + 5
        order = torch.randperm(pages, generator=host)
        table = torch.zeros(len(per), max(per), dtype=torch.int64)
        at = torch.cumsum(torch.tensor([0] + per), 0)
        j = torch.arange(max(per))
        held = j[None] < torch.tensor(per)[:, None]
        table[held] = order[(at[:-1, None] + j[None])[held]]
        s["table"], s["lengths"] = table.int().cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
        s["pools"] = _values((2, pages, Hkv, page, D), dt, gen)
        T = sum(news)
        if kind == "append":
            s["qkv"] = _values((T, (Hq + 2 * Hkv) * D), dt, gen)
            s["inv_freq"] = _frequencies(case["dims"])
            s["rows"] = torch.cat([torch.full((n,), i) for i, n in enumerate(news)]).int().cuda()
            s["positions"] = torch.cat([torch.arange(a, a + n) for a, n in zip(had, news)]).int().cuda()
        else:
            s["q"] = _values((T, Hq, D), dt, gen)
            s["starts"] = torch.cumsum(torch.tensor([0] + news), 0).int().cuda()
            s["sinks"] = torch.randn(Hq, generator=gen, device="cuda") if case["sinks"] else None
        return s
    T, V, n = case["T"], case["V"], case["history"]
    s["logits"] = (3.0 * torch.randn((T, V), generator=gen, device="cuda")).to(dt)
    none = dict.fromkeys(("history", "history_lengths", "prompts", "repetition", "presence", "frequency", "bias_ids",
                          "bias", "mask"))
    s.update(none)
    if case["penalties"]:
        # some tokens come again and again, as words do
        u = torch.rand((T, n), generator=gen, device="cuda")
        s["history"] = (u ** 4 * V).int().clamp(max=V - 1)
        s["history_lengths"] = torch.tensor(_spread(T, n) if T > 1 else [n], dtype=torch.int32).cuda()
        s["prompts"] = s["history_lengths"] // 3
        s["repetition"] = 1.0 + 0.3 * torch.rand(T, generator=gen, device="cuda")
        s["presence"], s["frequency"] = (0.5 * torch.rand(T, generator=gen, device="cuda") for _ in range(2))
    if case["bias"]:
        s["bias_ids"] = torch.rand((T, V), generator=gen, device="cuda").argsort(-1)[:, :case["bias"]].int().contiguous()
        s["bias"] = torch.randn(s["bias_ids"].shape, generator=gen, device="cuda")
    if case["mask"]:
        # a grammar allows few tokens here and most of them there
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (T, _cdiv(V, 32)), generator=gen, device="cuda").int()
        s["mask"][::2] &= torch.randint(-2 ** 31, 2 ** 31, (1, _cdiv(V, 32)), generator=gen, device="cuda").int() & 0x01010101
    return s


# ---- one pass --------------------------------------------------------------------


def _heads(s):
    """The queries (keys and values) of a projection's rows."""
    c = s["case"]
    T, D = s["qkv"].shape[0], c["D"]
    if c["kind"] == "rotary":
        return s["qkv"][:, :c["H"] * D].view(T, c["H"], D)
    q, k, v = s["qkv"].split((c["Hq"] * D, c["Hkv"] * D, c["Hkv"] * D), 1)
    return q.view(T, -1, D), k.view(T, -1, D), v.view(T, -1, D)


def _run_own(s):
    import mlxcel_amd as mq

    c = s["case"]
    kind = c["kind"]
    if kind == "rotary":
        return mq.rotary(_heads(s), s["positions"], s["inv_freq"], interleaved=c["interleaved"], factor=c["factor"])
    if kind == "append":
        q, k, v = _heads(s)
        q = mq.rotary_append(q, k, v, s["pools"][0], s["pools"][1], s["table"], s["positions"], s["rows"],
                             s["inv_freq"], lengths=s["lengths"], interleaved=c["interleaved"], factor=c["factor"])
        return q, s["pools"]
    if kind == "chunk":
        return mq.paged_attention_chunk(s["q"], s["pools"][0], s["pools"][1], s["table"], s["lengths"], s["starts"],
                                        window=c["window"], softcap=c["softcap"], sinks=s["sinks"])
    return mq.adjust_logits(s["logits"], history=s["history"], history_lengths=s["history_lengths"],
                            prompts=s["prompts"], repetition=s["repetition"], presence=s["presence"],
                            frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"])


def _plain_rotary(x, s):
    c = s["case"]
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = (angle.cos() * c["factor"]).float(), (angle.sin() * c["factor"]).float()
    n = c["dims"]
    turned, rest = x[..., :n].float(), x[..., n:]
    if c["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :n // 2], turned[..., n // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned.to(x.dtype), rest), -1)


def _plain_chunk(s):
    c = s["case"]
    Hkv, D, page, G = c["Hkv"], c["D"], c["page"], c["Hq"] // c["Hkv"]
    news, had = _news(c)  # a program knows the lengths of its own batch
    out = torch.empty_like(s["q"])
    first = 0
    for b, (n, a) in enumerate(zip(news, had)):
        at = torch.arange(a + n, device="cuda")
        lo = max(0, a + 1 - c["window"]) if c["window"] else 0  # no token sees a key before it
        at = at[lo:]
        ids = s["table"][b].long()[at // page]
        k, v = (pool[ids, :, at % page].transpose(0, 1).float().contiguous() for pool in s["pools"])
        q = s["q"][first:first + n].view(n, Hkv, G, D).permute(1, 0, 2, 3).reshape(Hkv, n * G, D).float()
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
        if c["softcap"]:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        mine = a + torch.arange(n, device="cuda").repeat_interleave(G)[:, None]
        keep = at[None] <= mine
        if c["window"]:
            keep = keep & (at[None] > mine - c["window"])
        x = torch.where(keep[None], x, -math.inf)
        m = x.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            sink = s["sinks"].view(Hkv, 1, G).expand(Hkv, n, G).reshape(Hkv, n * G, 1)
            m = torch.maximum(m, sink)
        p = torch.exp(x - m)
        total = p.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            total = total + torch.exp(sink - m)
        o = (torch.matmul(p, v) / total).view(Hkv, n, G, D).permute(1, 0, 2, 3).reshape(n, c["Hq"], D)
        out[first:first + n] = o.to(out.dtype)
        first += n
    return out


def _plain_adjust(s):
    x = s["logits"].float()
    T, V = x.shape
    if s["history"] is not None:
        ids = s["history"].long()
        at = torch.arange(ids.shape[1], device=x.device)[None]
        live = at < s["history_lengths"][:, None]
        seen = torch.zeros((T, V), dtype=torch.int32, device=x.device)
        times = torch.zeros_like(seen)
        seen.scatter_add_(1, ids, live.int())
        times.scatter_add_(1, ids, (live & (at >= s["prompts"][:, None])).int())
        x = torch.where(seen > 0, torch.where(x > 0, x / s["repetition"][:, None], x * s["repetition"][:, None]), x)
        x = x - torch.where(times > 0, s["presence"][:, None] + s["frequency"][:, None] * times, 0.0)
    if s["bias"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        token = torch.arange(V, device=x.device)
        x = torch.where((s["mask"][:, token // 32] >> (token % 32)) & 1 != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "rotary":
        return _plain_rotary(_heads(s), s)
    if kind == "append":
        q, k, v = _heads(s)
        pos, page = s["positions"].long(), s["case"]["page"]
        at = s["table"][s["rows"].long(), pos // page].long()
        s["pools"][0][at, :, pos % page] = _plain_rotary(k, s)
        s["pools"][1][at, :, pos % page] = v
        return _plain_rotary(q, s), s["pools"]
    if kind == "chunk":
        return _plain_chunk(s)
    return _plain_adjust(s)


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    """Bytes: each input read once, each output written once; operations of the products and sums."""
    kind, e = case["kind"], _SIZES[case["dtype"]]
    if kind == "rotary":
        n = case["T"] * case["H"]
        return {"bytes": 2 * n * case["D"] * e + 4 * case["T"] + 2 * case["dims"], "flops": 3 * n * case["dims"]}
    if kind == "append":
        T, heads = sum(_news(case)[0]), case["Hq"] + case["Hkv"]
        return {"bytes": 2 * T * (heads + case["Hkv"]) * case["D"] * e + 12 * T + 2 * case["dims"],
                "flops": 3 * T * heads * case["dims"]}
    if kind == "chunk":
        keys, pairs = _seen(case)
        T = sum(_news(case)[0])
        return {"bytes": 2 * keys * case["Hkv"] * case["D"] * e + 2 * T * case["Hq"] * case["D"] * e
                + 4 * keys / case["page"], "flops": 4 * pairs * case["Hq"] * case["D"]}
    T, V = case["T"], case["V"]
    lengths = (_spread(T, case["history"]) if T > 1 else [case["history"]]) if case["penalties"] else [0]
    return {"bytes": 2 * T * V * e + 4 * sum(lengths) + 8 * T * case["bias"] + (T * V / 8 if case["mask"] else 0),
            "flops": T * (V if case["mask"] else 0) + 4 * sum(lengths) + T * case["bias"]}


# ---- 64-bit results ------------------------------------------------------------------


def _exact_rotary(x, s):
    """Pairs as complex numbers times factor * exp(i angle), whole turns taken off the angle first."""
    c = s["case"]
    n, x = c["dims"], x.double()
    turns = s["positions"].double()[:, None] * (s["inv_freq"].double() / (2 * math.pi))[None]
    by = torch.polar(torch.full_like(turns, c["factor"]), 2 * math.pi * (turns - turns.round()))[:, None]
    out = x.clone()
    first, second = (slice(0, n, 2), slice(1, n, 2)) if c["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_chunk(s):
    """One head at a time, tokens in blocks: every token over its own range of keys."""
    c = s["case"]
    G, page = c["Hq"] // c["Hkv"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, length in enumerate(lengths):
        pos = torch.arange(length, device="cuda")
        ids = s["table"][b].long()[pos // page]
        for h in range(c["Hkv"]):
            k, v = (pool[ids, h, pos % page].double() for pool in s["pools"])
            for t0 in range(starts[b], starts[b + 1], 512):
                t1 = min(t0 + 512, starts[b + 1])
                end = length - starts[b + 1] + torch.arange(t0, t1, device="cuda") + 1
                q = s["q"][t0:t1, h * G:(h + 1) * G].double()
                x = (q.reshape(-1, c["D"]) @ k.t() / math.sqrt(c["D"])).view(t1 - t0, G, length)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                hidden = pos[None] >= end[:, None]
                if c["window"]:
                    hidden |= pos[None] < end[:, None] - c["window"]
                x.masked_fill_(hidden[:, None], -math.inf)
                if s["sinks"] is not None:
                    sink = s["sinks"][h * G:(h + 1) * G].double()[None, :, None].expand(t1 - t0, G, 1)
                    x = torch.cat([x, sink], -1)
                p = torch.softmax(x, -1)[..., :length]
                out[t0:t1, h * G:(h + 1) * G] = (p.reshape(-1, length) @ v).view(t1 - t0, G, c["D"])
    return out


def _exact_adjust(s):
    out = s["logits"].double()
    V = out.shape[1]
    for t, x in enumerate(out):
        if s["history"] is not None:
            n, p = int(s["history_lengths"][t]), int(s["prompts"][t])
            rep = s["repetition"][t].double()
            all_ids = torch.unique(s["history"][t, :n].long())
            x[all_ids] = torch.where(x[all_ids] > 0, x[all_ids] / rep, x[all_ids] * rep)
            ids, times = torch.unique(s["history"][t, p:n].long(), return_counts=True)
            x[ids] -= s["presence"][t].double() + s["frequency"][t].double() * times
        if s["bias"] is not None:
            x[s["bias_ids"][t].long()] += s["bias"][t].double()
        if s["mask"] is not None:
            bits = (s["mask"][t].long()[:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.reshape(-1)[:V] == 0] = -math.inf
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(_heads(s), s)
    if kind == "append":
        q, k, v = _heads(s)
        pools, page = s["pools"].double(), case["page"]
        k = _exact_rotary(k, s)
        for r in range(case["R"]):
            mine = torch.nonzero(s["rows"] == r)[:, 0]
            pos = s["positions"][mine].long()
            at = s["table"][r].long()[pos // page]
            pools[0, at, :, pos % page] = k[mine]
            pools[1, at, :, pos % page] = v[mine].double()
        return _exact_rotary(q, s), pools
    return _exact_chunk(s) if kind == "chunk" else _exact_adjust(s)
