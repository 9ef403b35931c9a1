"""The 8-bit block cache in 64 bits on the CPU: what the kernels of ``libleankv_bytes.so`` are compared with.

Written from the format's definition (``include/leankv_bytes.h``): blocks of 16 tokens of one sequence and kv head, codes ``rint(x 2^-e)``,
e the smallest whole number >= -126 with ``|x| <= 127 * 2^e``; a token that joins may raise e, and the codes that are there are rounded again.
"""

from __future__ import annotations

import math

import torch

BLOCK = 16
LARGEST = 2.0 ** 126


def least_exponent(amax: float, most: int) -> int:
    """The smallest whole e >= -126 with ``amax <= most * 2^e``."""
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax)[1] - 1 - (most + 1).bit_length() + 1)
        while amax > math.ldexp(most, e):
            e += 1
    return e


class Block:
    """Keys or values of up to 16 tokens of one kv head; ``scale_exp`` None: no number."""

    def __init__(self, dim: int):
        self.codes = torch.zeros(0, dim, dtype=torch.float64)
        self.scale_exp: int | None = -126

    def join(self, x: torch.Tensor) -> None:
        """New tokens [n, dim] (double) behind those that are here."""
        n = len(self.codes)
        amax = float(x.abs().max()) if bool(torch.isfinite(x).all()) else math.inf
        if self.scale_exp is None or amax >= LARGEST:
            self.scale_exp = None
            self.codes = torch.zeros(n + len(x), x.shape[1], dtype=torch.float64)
            return
        e = max(self.scale_exp if n else -126, least_exponent(amax, 127))
        old = torch.round(self.codes * math.ldexp(1.0, self.scale_exp - e)) if n else self.codes
        self.codes = torch.cat([old, torch.round(x * math.ldexp(1.0, -e))])
        self.scale_exp = e

    def values(self) -> torch.Tensor:
        if self.scale_exp is None:
            return torch.full_like(self.codes, math.nan)
        return self.codes * math.ldexp(1.0, self.scale_exp)


class Cache:
    """Sequences of one layer: ``blocks[which][sequence][head]`` is a list of blocks."""

    def __init__(self, batch: int, heads: int, dim: int):
        self.dim, self.heads = dim, heads
        self.blocks = [[[[] for _ in range(heads)] for _ in range(batch)] for _ in range(2)]
        self.n = [0] * batch

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """[B', H, T, D] for the first B' sequences."""
        for which, x in enumerate((k, v)):
            x = x.detach().cpu().double()
            for b in range(x.shape[0]):
                for h in range(self.heads):
                    row, at = self.blocks[which][b][h], 0
                    while at < x.shape[2]:
                        slot = (self.n[b] + at) % BLOCK
                        if slot == 0:
                            row.append(Block(self.dim))
                        take = min(BLOCK - slot, x.shape[2] - at)
                        row[-1].join(x[b, h, at:at + take])
                        at += take
        for b in range(k.shape[0]):
            self.n[b] += k.shape[2]

    def crop(self, n: int) -> None:
        for b in range(len(self.n)):
            if self.n[b] <= n:
                continue
            self.n[b] = n
            for which in range(2):
                for row in self.blocks[which][b]:
                    del row[-(-n // BLOCK):]
                    if n % BLOCK:
                        row[-1].codes = row[-1].codes[:n % BLOCK]

    def codes(self, b: int, which: int) -> torch.Tensor:
        """[H, T, D], whole numbers in double."""
        return torch.stack([torch.cat([x.codes for x in row]) for row in self.blocks[which][b]])

    def scales(self, b: int, which: int) -> torch.Tensor:
        return torch.tensor([[math.nan if x.scale_exp is None else math.ldexp(1.0, x.scale_exp) for x in row] for row in self.blocks[which][b]],
                            dtype=torch.float64)

    def values(self, b: int, which: int) -> torch.Tensor:
        return torch.stack([torch.cat([x.values() for x in row]) for row in self.blocks[which][b]])

    def attend(self, b: int, q: torch.Tensor, chosen: torch.Tensor | None = None) -> torch.Tensor:
        """Queries [Hq, T, D] of the sequence's last T tokens; ``chosen`` [H, K] blocks (-1: none) where only those are read."""
        q = q.detach().cpu().double()
        out = torch.zeros_like(q)
        group, n = q.shape[0] // self.heads, self.n[b]
        if n == 0:
            return out
        k, v = self.values(b, 0), self.values(b, 1)
        first = n - q.shape[1]                          # position of the first query
        for hq in range(q.shape[0]):
            h = hq // group
            if chosen is not None:
                at = torch.cat([torch.arange(BLOCK * j, min(BLOCK * j + BLOCK, n)) for j in chosen[h].tolist() if j >= 0])
                w = torch.softmax(q[hq] @ k[h, at].T / math.sqrt(self.dim), -1)
                out[hq] = w @ v[h, at]
                continue
            for t in range(max(0, -first), q.shape[1]):                # what nobody sees does not enter, not even as 0 * NaN
                w = torch.softmax(k[h, :first + t + 1] @ q[hq, t] / math.sqrt(self.dim), 0)
                out[hq, t] = w @ v[h, :first + t + 1]
        return out

    def choose(self, b: int, q: torch.Tensor, blocks: int, sinks: int, recent: int) -> torch.Tensor:
        """int32 [H, blocks]: what a query token [Hq, D] reads, ascending, then -1."""
        q = q.detach().cpu().double().view(self.heads, -1, self.dim)
        have = -(-self.n[b] // BLOCK)
        out = torch.full((self.heads, blocks), -1, dtype=torch.int32)
        for h in range(self.heads):
            picked = list(range(have))
            if have > blocks:
                amax = float(q[h].abs().max())
                i = torch.round(q[h] * math.ldexp(1.0, -least_exponent(amax, 2047))) if math.isfinite(amax) else torch.zeros_like(q[h])
                up, low = i.clamp(min=0).sum(0), i.clamp(max=0).sum(0)
                scores = []
                for j in range(sinks, have - recent):
                    block = self.blocks[0][b][h][j]
                    u = float((up * block.codes.amax(0) + low * block.codes.amin(0)).sum())
                    value = math.inf if block.scale_exp is None else float(torch.tensor(u, dtype=torch.float32)) * math.ldexp(1.0, block.scale_exp)
                    scores.append((-float(torch.tensor(value, dtype=torch.float64).float()), j))
                picked = sorted([*range(sinks), *(j for _, j in sorted(scores)[:blocks - sinks - recent]), *range(have - recent, have)])
            out[h, :len(picked)] = torch.tensor(picked, dtype=torch.int32)
        return out
