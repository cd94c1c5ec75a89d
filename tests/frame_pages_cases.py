"""Calls of attention over pages that are shared out in ways which small calls are not, and what it takes to
make and to check them: caches of random codes, and the definition for some of a call's sequences and heads.

A case: (type, head size, q heads, kv heads, page, prefix, query lengths, own lengths, frame, back, ahead, sinks)."""
from __future__ import annotations

import math

import torch

import frame_attention_reference as ref
import frame_mx_reference as mx

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BITS = [0, 8, 4]  # 0: pages of the type
GAP = 2  # rows of no sequence in front; one more behind


def scaled(case, bits):
    """As many bytes of a prefix, whatever the bits of a key: its tokens and the window's frames grow."""
    times = 16 // (bits or 16)
    back = case[9] if case[9] < 0 else case[9] * times
    return case[:5] + (case[5] * times,) + case[6:9] + (back,) + case[10:]


# Prefixes that are read once for all sequences (in 16 bits; others: scaled): (the rows of a block of the
# prefix and of the sequences' own, case).
READ_ONCE = [
    ((128, 16), ("bf16", 64, 8, 2, 64, 8100, [1] * 64, [1 + 7 * s % 90 for s in range(64)], 1, -1, 0, 0)),
    ((128, 16), ("bf16", 128, 4, 1, 16, 4100, [1] * 70, [1 + 5 * s % 40 for s in range(70)], 1, -1, 0, 0)),
    ((128, 16), ("f16", 64, 8, 4, 32, 4000, [1] * 66, [1 + 3 * s % 50 for s in range(66)], 1, 3500, 0, 2)),  # a window that ends in the prefix
    ((128, 16), ("f16", 128, 8, 4, 8, 3000, [3 if s % 4 else 0 for s in range(40)], [s % 7 for s in range(40)], 1, -1, 0, 0)),  # queries past their own keys
    ((128, 16), ("f16", 64, 4, 4, 64, 6000, [0 if s % 5 == 3 else 1 for s in range(150)], [s % 3 for s in range(150)], 7, 600, 0, 3)),
    ((32, 16), ("f16", 128, 8, 8, 8, 2200, [1] * 16, [2 + s for s in range(16)], 1, -1, 0, 0)),
    ((16, 16), ("bf16", 64, 8, 8, 64, 8500, [1] * 8, [4 + s for s in range(8)], 1, -1, 0, 0)),
    ((128, 32), ("bf16", 64, 12, 2, 16, 6500, [2 + s % 3 for s in range(48)], [7 * s % 40 for s in range(48)], 5, 1200, 1, 1)),
    ((128, 32), ("f16", 128, 8, 2, 64, 5400, [5] * 24, [5 + s for s in range(24)], 1, -1, -1, 0)),
    ((128, 128), ("bf16", 64, 8, 8, 16, 1000, [33 + s % 9 for s in range(130)], [40 + 31 * s % 300 for s in range(130)], 16, -1, 0, 0)),
    ((128, 128), ("f16", 128, 12, 4, 16, 2300, [s % 12 for s in range(80)], [s % 12 + s for s in range(80)], 1, -1, 0, 0)),
]

# Blocks of 128 rows over the sequences' own keys, a private prefix before them or none.
TILES = [
    # Four blocks, the last with sixteen rows; window, sinks, frames that end inside tiles; queries without keys.
    ("bf16", 64, 16, 8, 16, 0, [200 - s for s in range(33)], [1 + 61 * s % 500 for s in range(33)], 50, 3, 0, 1),
    ("f16", 64, 16, 8, 64, 0, [200 - 5 * s for s in range(33)], [210 + 61 * s % 300 for s in range(33)], 1, 90, 0, 70),
    # Long keys, and short ones beside them.
    ("bf16", 64, 16, 8, 64, 0, [200] + [150] * 8, [8300] + [150 + s for s in range(8)], 1, -1, 0, 0),
    ("f16", 64, 16, 8, 8, 0, [200] + [150] * 8, [8300] + [150 + s for s in range(8)], 64, 126, 1, 2),
    ("bf16", 128, 24, 8, 16, 0, [40 - s for s in range(33)], [61 * s % 300 for s in range(33)], 7, 9, 0, 2),
    ("f16", 128, 8, 8, 64, 0, [500, 0, 1] + [390] * 6, [500, 70, 1] + [400 + s for s in range(6)], 64, 1, 0, 1),
    ("bf16", 128, 16, 8, 8, 0, [250] * 9, [260 + 40 * s for s in range(9)], 1, -1, -1, 0),
    # A prefix of their own reading: rows that fill blocks, or little to read again.
    ("f16", 64, 16, 8, 16, 300, [200 - s for s in range(33)], [1 + 61 * s % 300 for s in range(33)], 50, 5, 0, 1),
    ("bf16", 128, 24, 8, 8, 77, [40 - s for s in range(33)], [61 * s % 200 for s in range(33)], 1, -1, 0, 0),
    ("f16", 128, 8, 8, 64, 700, [500, 0, 1] + [390] * 6, [500, 70, 1] + [400 + s for s in range(6)], 64, 8, 0, 1),
]


def name_of(case):
    return f"{case[0]}-d{case[1]}-h{case[2]}.{case[3]}-p{case[4]}-P{case[5]}-n{len(case[6])}-q{max(case[6])}-k{max(case[7])}-f{case[8]}w{case[9]}a{case[10]}s{case[11]}"


def rows_of(case):
    """Rows of the queries' tensor."""
    return GAP + sum(case[6]) + 1


class Call:
    """A cache, queries and outputs of one case, on the GPU; the cache's buffers on the CPU too."""

    def __init__(self, case, bits, seed=1):
        self.case, self.bits = case, bits
        name, dim, hq, hk, page, prefix, nq, nk = case[:8]
        dtype, g = DTYPES[name], torch.Generator().manual_seed(seed)
        self.cu = [GAP]
        for n in nq:
            self.cu.append(self.cu[-1] + n)
        self.q = torch.randn(rows_of(case), hq, dim, generator=g).to(dtype)
        used = [-(-n // page) for n in [prefix] + nk]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.prefix_table = order[:used[0]].clone()
        self.table = torch.full((len(nk), max(max(used[1:]), 1) + 1), -1, dtype=torch.int32)
        at = used[0]
        for row, n in zip(self.table, used[1:]):
            row[:n] = order[at:at + n]
            at += n
        if bits:  # magnitudes up to 7 (8 bits) and 3 (4 bits), NaN's code not among them
            codes = [torch.randint(0, 256, (pages, hk, page, dim * bits // 8), generator=g, dtype=torch.uint8) for _ in range(2)]
            if bits == 8:
                codes = [c - ((c & 127) == 127).to(torch.uint8) for c in codes]
            low = 117 if bits == 8 else 122
            scales = [torch.randint(low, low + 5, (pages, hk, page, dim // 32), generator=g, dtype=torch.uint8) for _ in range(2)]
            self.buffers = codes + scales
        else:
            self.buffers = [torch.randn(pages, page, hk, dim, generator=g).to(dtype) for _ in range(2)]

    def run(self, fa, ctx, buffers=None, prefix_table=None, table=None):
        name, dim, hq, hk, page, prefix, nq, nk, *window = self.case
        i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
        on = [b.cuda() for b in (buffers or self.buffers)]
        out = torch.full(self.q.shape, float("nan"), dtype=self.q.dtype, device="cuda")
        lse = torch.full(self.q.shape[:2], float("nan"), device="cuda")
        fa.FrameAttention(ctx, hq, hk, dim, *window).shared_dev(
            self.q.cuda(), fa.MxPages(*on) if self.bits else tuple(on), (self.prefix_table if prefix_table is None else prefix_table).cuda(),
            i32([prefix]), (self.table if table is None else table).cuda(), i32(self.cu), i32(nk), out, lse, max_q=max(nq), max_kv=max(nk),
            max_prefix=prefix)
        torch.cuda.synchronize()
        return out.cpu(), lse.cpu()

    def seen(self, s):
        """[queries][keys] of sequence s, its prefix's keys first."""
        prefix, frame, back, ahead, sinks = self.case[5], *self.case[8:]
        nq, nk = self.case[6][s], self.case[7][s]
        p = (prefix + nk - nq + torch.arange(nq))[:, None]
        f, fj = torch.div(p, frame, rounding_mode="floor"), (torch.arange(prefix + nk) // frame)[None]
        return (p >= 0) & ((fj <= f + ahead) | (ahead < 0)) & ((fj >= f - back) | (back < 0) | (fj < sinks))

    def rows(self, table, n, head, part):
        """[n][dim] in 64 bits: the first n keys (part 0) or values of a table and one key head."""
        at = torch.arange(n)
        page, which = self.case[4], table[at // self.case[4]].long()
        if not self.bits:
            return self.buffers[part][which, at % page, head].double()
        return mx.values(self.buffers[part][which, head, at % page], self.buffers[2 + part][which, head, at % page], self.bits)

    def place(self, s, j):
        """(page, token of the page) of key j of sequence s, the prefix's first."""
        prefix, page = self.case[5], self.case[4]
        return (int(self.prefix_table[j // page]), j % page) if j < prefix else (int(self.table[s][(j - prefix) // page]), (j - prefix) % page)

    def spoiled(self, page, token, part):
        """Buffers in which a key's (part 0) or value's first block of every head reads as NaN."""
        bad = [b.clone() for b in self.buffers]
        if self.bits:
            bad[2 + part][page, :, token, 0] = 255
        else:
            bad[part][page, token, :, 0] = float("nan")
        return bad

    def sequences(self, most=6):
        """Some of the sequences that have queries: the first and last, the longest, the shortest, and between."""
        nq, nk = self.case[6:8]
        have = [s for s in range(len(nq)) if nq[s]]
        some = {have[0], have[-1], max(have, key=lambda s: nk[s]), min(have, key=lambda s: nk[s]), max(have, key=lambda s: nq[s] - nk[s])}
        return sorted(some | set(have[:: max(1, len(have) // most)][:most]))

    def compare(self, out, lse, gone=None):
        """Some sequences and heads against the definition, within the bounds on roundings; every row of a
        sequence was written, and no other. gone: the pages that are not there, by sequence (-1: the prefix's)."""
        name, dim, hq, hk, page, prefix, nq, nk, *_ = self.case
        mine = torch.zeros(len(self.q), dtype=torch.bool)
        mine[self.cu[0]:self.cu[-1]] = True
        assert torch.isnan(out[~mine]).all() and torch.isnan(lse[~mine]).all(), "rows of no sequence were written"
        assert torch.isfinite(out[mine]).all() and not torch.isnan(lse[mine]).any()
        group = hq // hk
        for s in self.sequences():
            rows, seen = slice(self.cu[s], self.cu[s + 1]), self.seen(s)
            for first, end, of in ((0, prefix, -1), (prefix, prefix + nk[s], s)):
                for p in (gone or {}).get(of, ()):
                    seen[:, first + p * page:min(first + (p + 1) * page, end)] = False
            for h in {(5 * s + 1) % hq, hq - 1 - s % group}:
                keys, values = (torch.cat([self.rows(self.prefix_table, prefix, h // group, part), self.rows(self.table[s], nk[s], h // group, part)])
                                for part in range(2))
                want = ref.attention(self.q[rows, h], keys, values, seen, 1 / math.sqrt(dim), self.q.dtype)
                for what, got in (("out", out[rows, h]), ("lse", lse[rows, h])):
                    exact, bound = want[what]
                    got, fine = got.double(), torch.isfinite(exact)
                    assert torch.equal(fine, torch.isfinite(got)), (what, s, h)
                    if fine.any():
                        off = ((got - exact).abs()[fine] / (bound[fine] + 1e-30)).max().item()
                        assert off <= 1.0, (what, s, h, off)

    def unseen(self, fa, ctx, out, lse, s, j, **tables):
        """NaN in key j of sequence s (the prefix's: of all sequences), then in its value: rows that do not see
        it have the bits that they had, those that do have NaN."""
        sees = torch.zeros(len(self.q), dtype=torch.bool)
        for t in range(len(self.cu) - 1) if j < self.case[5] else (s,):
            sees[self.cu[t]:self.cu[t + 1]] = self.seen(t)[:, j]
        rest = torch.zeros_like(sees)
        rest[self.cu[0]:self.cu[-1]] = True
        rest &= ~sees
        for part in range(2):
            got, got_lse = self.run(fa, ctx, self.spoiled(*self.place(s, j), part), **tables)
            assert torch.equal(got[rest], out[rest]) and torch.equal(got_lse[rest], lse[rest]), (s, j, part)
            assert torch.isnan(got[sees]).any(-1).all() and (part or torch.isnan(got[sees]).all()), (s, j, part)
