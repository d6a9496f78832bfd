"""A cache of pages, and attention over it, in float64 on the CPU: slot by slot
and key by key from the definitions, for tests."""

from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn


def codes_of(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 magnitudes, by the list of all of them; ties to even codes,
    saturating; what is not finite becomes NaN."""
    grid = torch.tensor([m * 2.0**-9 for m in range(8)] +
                        [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119],
                        dtype=torch.float64)
    a = x.abs().clamp(max=448.0).nan_to_num(0.0)
    up = torch.searchsorted(grid, a.contiguous()).clamp(max=126)
    down = (up - 1).clamp(min=0)
    above, below = grid[up] - a, a - grid[down]
    pick = torch.where((below < above) | ((below == above) & (down % 2 == 0)), down, up)
    return torch.where(torch.isfinite(x), torch.copysign(grid[pick], x), torch.full_like(x, float("nan")))


def least_exponent(x: torch.Tensor) -> int:
    """Least e with 448 * 2**e >= max |x| over the finite values."""
    x = x[torch.isfinite(x)].abs()
    top = float(x.max()) if x.numel() else 0.0
    e = -110
    while e < 119 and 448.0 * 2.0**e < top:
        e += 1
    return e


class Pool:
    """One tensor of a pool: codes (or values) in float64, exponents as ints."""

    def __init__(self, pool: torch.Tensor, exponent: torch.Tensor | None):
        self.data = pool.detach().cpu().double()
        self.exponent = None if exponent is None else exponent.detach().cpu().long()

    def write(self, page: int, lo: int, rows: torch.Tensor) -> None:
        """New tokens rows (heads, n, D) at slots lo .. of a page."""
        n = rows.shape[1]
        if self.exponent is None:
            self.data[page, :, lo:lo + n] = rows
            return
        for h in range(rows.shape[0]):
            e, old = least_exponent(rows[h]), int(self.exponent[page, h])
            if lo > 0:
                e = max(e, old)
                if e > old:
                    self.data[page, h] = codes_of(self.data[page, h] * 2.0 ** (old - e))
            self.data[page, h, lo:lo + n] = codes_of(rows[h] / 2.0**e)
            self.exponent[page, h] = e

    def values(self) -> torch.Tensor:
        if self.exponent is None:
            return self.data
        return self.data * torch.exp2(self.exponent.double())[:, :, None, None]


def append(pool: Pool, x, block_table, lengths, counts) -> None:
    """x (B, H, L, D) float64; the tables as lists."""
    pages, _, size, _ = pool.data.shape
    for b in range(x.shape[0]):
        count = max(0, min(counts[b], x.shape[2]))
        first = lengths[b] - count
        by_block: dict[int, list[int]] = {}
        for i in range(count):
            p = first + i
            if p >= 0 and p // size < len(block_table[b]) and 0 <= block_table[b][p // size] < pages:
                by_block.setdefault(p // size, []).append(i)
        for block, tokens in by_block.items():
            pool.write(block_table[b][block], (first + tokens[0]) % size, x[b, :, tokens])


def rotate(x, cos, sin, start, half):
    """Channels [start, start + 2P) of x (B, H, L, D) in float64."""
    P = cos.shape[-1]
    x = x.double().clone()
    y = x[..., start:start + 2 * P]
    a, b = (y[..., :P], y[..., P:]) if half else (y[..., 0::2], y[..., 1::2])
    c, s = cos.double(), sin.double()
    u, v = a * c - b * s, a * s + b * c
    x[..., start:start + 2 * P] = torch.cat([u, v], -1) if half else torch.stack([u, v], -1).flatten(-2)
    return x


def attend(q, key: torch.Tensor, value: torch.Tensor, block_table, lengths, counts, *, window=0, cap=0.0, slopes=None,
           scale=None):
    """(out, lse, spread, score): q (B, Hq, Lq, D) float64 against pools of values
    (pages, H, size, D); spread: sum of p |v| / sum of p, score: the largest sum of
    |q_c k_c| * scale of a row's keys plus its largest |changed score|."""
    B, Hq, Lq, D = q.shape
    pages, H, size, _ = key.shape
    scale = D**-0.5 if scale is None else scale
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((B, Hq, Lq), float("-inf"), dtype=torch.float64)
    score = torch.zeros((B, Hq, Lq), dtype=torch.float64)
    for b in range(B):
        count = max(0, min(counts[b], Lq))
        last = max(lengths[b], 0)
        n = min(last, len(block_table[b]) * size)
        has = torch.tensor([0 <= block_table[b][j // size] < pages for j in range(n)], dtype=torch.bool)
        at = [(block_table[b][j // size] if has[j] else 0, j % size) for j in range(n)]
        if n == 0:
            continue
        pg, sl = torch.tensor([a[0] for a in at]), torch.tensor([a[1] for a in at])
        j, i = torch.arange(n), torch.arange(Lq)
        distance = (last - count + i)[:, None] - j
        seen = has & (distance >= 0) & (i < count)[:, None]
        if window:
            seen &= distance < window
        rows = seen.any(1)  # the others have no key
        for h in range(Hq):
            # Values that no row sees may be anything.
            used = seen.any(0)
            k, v = (torch.where(used[:, None], t[pg, h * H // Hq, sl], 0.0) for t in (key, value))
            z = scale * (q[b, h] @ k.T)
            mag = scale * (q[b, h].abs() @ k.T.abs())
            if cap:
                z = cap * torch.tanh(z / cap)
            if slopes is not None:
                z = z - float(slopes[h]) * distance.double()
            z = z.masked_fill(~seen, float("-inf"))[rows]
            w = torch.softmax(z, 1)
            out[b, h, rows] = w @ v
            spread[b, h, rows] = w @ v.abs()
            lse[b, h, rows] = torch.logsumexp(z, 1)
            score[b, h, rows] = mag.masked_fill(~seen, 0.0)[rows].amax(1) + z.amax(1).abs() + 1.0
    return out, lse, spread, score
