"""Decoding with a paged cache: quantized projections, rotated appends, paged
attention of prompts and single tokens, cache pages, residual norms, logit
adjustments and token log probabilities together.

    python examples/paged_decode.py

A random-weight decoder answers prompts of several lengths.  The prompts are read
once, a chunk of each at a time, then forked into one sequence per candidate
first token (the alternatives of `token_logprobs`); the sequences share the
prompt's full pages.  Each step reserves a page where a sequence needs one,
rotates the step's queries and keys, appends the keys and values and attends to
the cache; tokens that were there already may be penalized; the log
probabilities of what was chosen rank the answers.  Finished sequences are freed, and the pages that are left moved to the
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
        self.inv_freq, _ = mq.rotary_frequencies(hd)
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

    def forward(self, tokens, positions, rows, attend):
        """Hidden states of tokens at `positions` of the cache's `rows`, which have room for them;
        attend(q, keys, values) is the attention over a layer's pools."""
        n_layers = len(self.layers)
        h = self.embed[tokens]
        h, x = mq.residual_norm(h, h, scale=0.0, pre_weight=self.layers[0]["pre"])  # the first norm alone
        for i, L in enumerate(self.layers):
            q, k, v = (t.view(len(x), -1, self.hd) for t in self.project(x, L["qkv"]))
            kp, vp = self.pools[i], self.pools[n_layers + i]
            q = mq.rotary_append(q, k, v, kp, vp, self.table, positions, rows, self.inv_freq, lengths=self.lengths)
            a = attend(q, kp, vp)
            y = mq.quantized_matmul(a.view(len(x), -1), *L["o"], True, GS, BITS)
            h, x = mq.residual_norm(h, y, post_weight=L["post"], pre_weight=L["mid"])
            g, u = self.project(x, L["gu"])
            y = mq.quantized_matmul((torch.nn.functional.silu(g.float()) * u.float()).to(x.dtype), *L["d"], True, GS, BITS)
            nxt = self.layers[i + 1]["pre"] if i + 1 < n_layers else self.last
            h, x = mq.residual_norm(h, y, pre_weight=nxt)
        return x

    def step(self, tokens, live):
        """One token for each row where `live` (others are left alone): logits [rows, vocab].

        A row that the cache has no page for stays as it was; `granted` says so."""
        positions = torch.where(live, self.lengths, -1)
        granted = mq.cache_reserve(self.table, self.lengths, self.refs, live.int(), self.page)
        x = self.forward(tokens, positions, self.rows,
                         lambda q, kp, vp: mq.paged_attention(q, kp, vp, self.table, self.lengths))
        return mq.quantized_matmul(x, *self.lm, True, GS, BITS), granted

    def read(self, prompts, chunk=64):
        """Appends prompt i (a list of tokens) to row i, up to `chunk` tokens of each at a time:
        the logits after each one's last token."""
        n, dev, done, logits = len(prompts), "cuda", [0] * len(prompts), [None] * len(prompts)
        had = self.lengths[:n].tolist()
        while any(d < len(p) for d, p in zip(done, prompts)):
            new = [min(chunk, len(p) - d) for d, p in zip(done, prompts)]
            ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
            starts = [0]
            for m in new:
                starts.append(starts[-1] + m)
            rows = ints([i for i, m in enumerate(new) for _ in range(m)])
            positions = ints([had[i] + done[i] + j for i, m in enumerate(new) for j in range(m)])
            tokens = [t for d, m, p in zip(done, new, prompts) for t in p[d:d + m]]
            counts = ints(new + [0] * (len(self.rows) - n))
            if not bool(mq.cache_reserve(self.table, self.lengths, self.refs, counts, self.page).all()):
                raise RuntimeError("the cache has no page left")
            at = ints(starts)
            x = self.forward(torch.tensor(tokens, device=dev), positions, rows, lambda q, kp, vp: mq.paged_attention_chunk(
                q, kp, vp, self.table[:n], self.lengths[:n], at))
            done = [d + m for d, m in zip(done, new)]
            ends = [i for i, m in enumerate(new) if m and done[i] == len(prompts[i])]
            if ends:
                out = mq.quantized_matmul(x[[starts[i + 1] - 1 for i in ends]], *self.lm, True, GS, BITS)
                for i, row in zip(ends, out):
                    logits[i] = row
        return torch.stack(logits)

    def answer(self, prompts, ways=3, steps=12, chunk=64, repetition=1.0):
        """For each prompt (a list of tokens) `ways` answers of `steps` tokens that
        begin with its most probable first tokens and go on greedily: a list of
        (prompt index, tokens, sum of their log probabilities).  Before each choice
        after the first the logits of tokens that the prompt or the answer has are
        divided by `repetition` (multiplied where negative)."""
        n, dev = len(prompts), "cuda"
        need = n * (1 + ways)
        if need > len(self.rows):
            raise ValueError(f"{need} sequences do not fit the table's {len(self.rows)} rows")
        first = self.read(prompts, chunk)
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
        if repetition != 1.0:
            # what each answer's choice looks back on: the prompt, then the answer
            longest = max(map(len, prompts))
            history = torch.zeros(n * ways, longest + steps, dtype=torch.int32, device=dev)
            for i, p in enumerate(prompts):
                history[i * ways:(i + 1) * ways, :len(p)] = torch.tensor(p, dtype=torch.int32, device=dev)
            seen = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev).repeat_interleave(ways)
            penalty = torch.full((n * ways,), repetition, device=dev)
            each = torch.arange(n * ways, device=dev)
        for _ in range(steps - 1):
            tokens[n:n + n * ways] = answers[-1].long()
            out, granted = self.step(tokens, live)
            if not bool(granted.all()):
                raise RuntimeError("the cache has no page left")
            out = out[n:n + n * ways]
            if repetition != 1.0:
                history[each, seen.long()] = answers[-1]
                seen = seen + 1
                choice = mq.adjust_logits(out, history=history, history_lengths=seen, repetition=penalty)
                _, _, _, ids = mq.token_logprobs(choice, answers[-1][:, None].contiguous(), top_k=1)
                given, _ = mq.token_logprobs(out, ids.contiguous())[:2]
            else:
                _, _, given, ids = mq.token_logprobs(out, answers[-1][:, None].contiguous(), top_k=1)
            answers.append(ids[:, 0].contiguous())
            score = score + given[:, 0]
        mq.cache_free(self.table, self.lengths, self.refs, dst, self.page)
        answers = torch.stack(answers, 1).tolist()
        return [(i // ways, a, s) for i, (a, s) in enumerate(zip(answers, score.tolist()))]


def main():
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 2000, (n,), generator=gen).tolist() for n in (5, 33, 17)]
    model = PagedDecoder()
    for i, tokens, score in model.answer(prompts, repetition=1.2):
        print(f"prompt {i} ({len(prompts[i])} tokens): {score:8.3f}  {tokens}")
    print(f"pages held at the end: {int((model.refs > 0).sum())}")


if __name__ == "__main__":
    main()
