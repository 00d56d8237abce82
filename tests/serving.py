"""Shared by the tests of the serving operators: caches dealt out at random,
tolerances."""
import numpy as np
import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


def within(got, want, slack, what=""):
    """|got - want| at most the slack and the rounding to got's type (half a
    step relative, half the smallest step near 0; infinity past its range)."""
    info = torch.finfo(got.dtype)
    g, want = f64(got), np.where(np.abs(want) > info.max, np.copysign(np.inf, want), want)
    bad = ~(np.abs(g - want) <= slack + info.eps / 2 * (np.abs(want) + slack) + info.tiny * info.eps / 2)
    bad &= ~((g == want) | (np.isnan(g) & np.isnan(want)))
    assert not bad.any(), (what, int(bad.sum()), g[bad][:4], want[bad][:4],
                           (np.abs(g - want) / (np.abs(want) + 1e-30))[bad][:4])


class Cache:
    """Random pools and a table whose pages are dealt out in random order; every
    slot that no sequence holds is NaN."""

    def __init__(self, lengths, Hkv, D, page, dtype, seed, spare=3, width=None, layout="pages"):
        g = torch.Generator().manual_seed(seed)
        per = [-(-max(n, 0) // page) for n in lengths]
        self.pages, self.page, self.D, self.Hkv = sum(per) + spare, page, D, Hkv
        self.width = max([1] + per) if width is None else width
        order = torch.randperm(self.pages, generator=g)
        self.table = np.full((len(lengths), self.width), -1, np.int32)
        at = 0
        held = torch.zeros(self.pages, page, dtype=torch.bool)
        for r, n in enumerate(per):
            self.table[r, :n] = order[at:at + n].numpy()
            for j in range(n):
                held[order[at + j], :min(page, lengths[r] - j * page)] = True
            at += n
        kv = []
        for _ in range(2):
            t = torch.randn(self.pages, Hkv, page, D, generator=g)
            t[~held[:, None, :].expand(-1, Hkv, -1)] = float("nan")
            kv.append(t.to(DTYPES[dtype]))
        if layout == "pages":
            self.k, self.v = (t.cuda() for t in kv)
        elif layout == "tokens":  # [pages, page, Hkv, D] in memory
            self.k, self.v = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in kv)
        else:  # keys and values in one allocation, rows padded by 2 elements
            both = torch.full((self.pages, 2, Hkv, page, D + 2), float("nan"), dtype=DTYPES[dtype])
            both[..., :D] = torch.stack(kv, 1)
            both = both.cuda()
            self.k, self.v = both[:, 0, ..., :D], both[:, 1, ..., :D]
        self.lengths = np.array(lengths, np.int32)
