"""Decoding with a paged cache: quantized projections, paged attention, cache
pages, residual norms and token log probabilities together.

    python examples/paged_decode.py

A random-weight decoder answers prompts of several lengths.  Each prompt is read
once, then forked into one sequence per candidate first token (the alternatives
of `token_logprobs`); the sequences share the prompt's full pages.  Each step
reserves a page where a sequence needs one, appends the step's keys and values
and attends to the cache; the log probabilities of what was chosen rank the
answers.  Finished sequences are freed, and the pages that are left moved to the
front of the pools.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import mlxcel_amd as mq  # noqa: E402

GS, BITS = 64, 4  # of the quantized weights


class PagedDecoder:
    def __init__(self, layers=3, hidden=512, nq=8, nkv=2, hd=64, inter=1024, vocab=2000, rows=16, width=16, pages=96,
                 page=16, seed=0):
        self.hidden, self.nq, self.nkv, self.hd, self.page = hidden, nq, nkv, hd, page
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def linear(n, k):
            return mq.quantize((torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5).to(torch.bfloat16), GS, BITS)

        def weight(n):
            return (1 + 0.1 * torch.randn(n, device="cuda", generator=gen)).to(torch.bfloat16)

        self.layers = [dict(qkv=[linear(nq * hd, hidden), linear(nkv * hd, hidden), linear(nkv * hd, hidden)],
                            o=linear(hidden, nq * hd), gu=[linear(inter, hidden), linear(inter, hidden)],
                            d=linear(hidden, inter), pre=weight(hidden), mid=weight(hidden), post=weight(hidden))
                       for _ in range(layers)]
        self.last, self.lm = weight(hidden), linear(vocab, hidden)
        self.embed = torch.randn(vocab, hidden, device="cuda", generator=gen).to(torch.bfloat16)
        # the cache: keys of every layer, then values; its book
        self.pools = [torch.zeros(pages, nkv, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2 * layers)]
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.rows = torch.arange(rows, dtype=torch.int32, device="cuda")
        inv = 10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        angle = torch.arange(width * page, device="cuda")[:, None] * inv
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def rope(self, x, positions):
        cos, sin = (t[positions.long().clamp(min=0)][:, None] for t in (self.cos, self.sin))
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)

    @staticmethod
    def project(x, ws):
        return mq.quantized_matmul_multi(x, [w[0] for w in ws], [w[1] for w in ws], [w[2] for w in ws], GS, BITS)

    def step(self, tokens, live):
        """One token for each row where `live` (others are left alone): logits [rows, vocab].

        A row that the cache has no page for stays as it was; `granted` says so."""
        positions = torch.where(live, self.lengths, -1)
        granted = mq.cache_reserve(self.table, self.lengths, self.refs, live.int(), self.page)
        n_layers = len(self.layers)
        h = self.embed[tokens]
        h, x = mq.residual_norm(h, h, scale=0.0, pre_weight=self.layers[0]["pre"])  # the first norm alone
        for i, L in enumerate(self.layers):
            q, k, v = self.project(x, L["qkv"])
            q, k = (self.rope(t.view(len(x), -1, self.hd), positions) for t in (q, k))
            kp, vp = self.pools[i], self.pools[n_layers + i]
            mq.cache_append(k, v.view(len(x), -1, self.hd), kp, vp, self.table, positions, self.rows,
                            lengths=self.lengths)
            a = mq.paged_attention(q, kp, vp, self.table, self.lengths)
            y = mq.quantized_matmul(a.view(len(x), -1), *L["o"], True, GS, BITS)
            h, x = mq.residual_norm(h, y, post_weight=L["post"], pre_weight=L["mid"])
            g, u = self.project(x, L["gu"])
            y = mq.quantized_matmul((torch.nn.functional.silu(g.float()) * u.float()).to(x.dtype), *L["d"], True, GS, BITS)
            nxt = self.layers[i + 1]["pre"] if i + 1 < n_layers else self.last
            h, x = mq.residual_norm(h, y, pre_weight=nxt)
        return mq.quantized_matmul(x, *self.lm, True, GS, BITS), granted

    def answer(self, prompts, ways=3, steps=12):
        """For each prompt (a list of tokens) `ways` answers of `steps` tokens that
        begin with its most probable first tokens and go on greedily: a list of
        (prompt index, tokens, sum of their log probabilities)."""
        n, dev = len(prompts), "cuda"
        need = n * (1 + ways)
        if need > len(self.rows):
            raise ValueError(f"{need} sequences do not fit the table's {len(self.rows)} rows")
        # the prompts, a position a step
        logits = [None] * n
        for t in range(max(map(len, prompts))):
            live = torch.zeros(len(self.rows), dtype=torch.bool)
            tokens = torch.zeros(len(self.rows), dtype=torch.int64)
            for i, p in enumerate(prompts):
                if t < len(p):
                    live[i], tokens[i] = True, p[t]
            out, granted = self.step(tokens.to(dev), live.to(dev))
            if not bool(granted.all()):
                raise RuntimeError("the cache has no page left")
            for i, p in enumerate(prompts):
                if t == len(p) - 1:
                    logits[i] = out[i]
        first = torch.stack(logits)
        _, _, top, ids = mq.token_logprobs(first, torch.zeros(n, 1, dtype=torch.int32, device=dev), top_k=ways)
        # a row for each answer; the prompt's own row goes
        src = torch.arange(n, dtype=torch.int32, device=dev).repeat_interleave(ways)
        dst = n + torch.arange(n * ways, dtype=torch.int32, device=dev)
        if not bool(mq.cache_fork(self.pools, self.table, self.lengths, self.refs, src, dst).all()):
            raise RuntimeError("the cache has no page left")
        mq.cache_free(self.table, self.lengths, self.refs, self.rows[:n], self.page)
        mq.cache_compact(self.pools, self.table, self.lengths, self.refs)
        answers, score = [ids.reshape(-1)], top.reshape(-1)
        live = (self.rows >= n) & (self.rows < n * (1 + ways))
        tokens = torch.zeros(len(self.rows), dtype=torch.int64, device=dev)
        for _ in range(steps - 1):
            tokens[n:n + n * ways] = answers[-1].long()
            out, granted = self.step(tokens, live)
            if not bool(granted.all()):
                raise RuntimeError("the cache has no page left")
            out = out[n:n + n * ways]
            _, _, top, ids = mq.token_logprobs(out, answers[-1][:, None].contiguous(), top_k=1)
            answers.append(ids[:, 0].contiguous())
            score = score + top[:, 0]
        mq.cache_free(self.table, self.lengths, self.refs, dst, self.page)
        answers = torch.stack(answers, 1).tolist()
        return [(i // ways, a, s) for i, (a, s) in enumerate(zip(answers, score.tolist()))]


def main():
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 2000, (n,), generator=gen).tolist() for n in (5, 33, 17)]
    model = PagedDecoder()
    for i, tokens, score in model.answer(prompts):
        print(f"prompt {i} ({len(prompts[i])} tokens): {score:8.3f}  {tokens}")
    print(f"pages held at the end: {int((model.refs > 0).sum())}")


if __name__ == "__main__":
    main()
