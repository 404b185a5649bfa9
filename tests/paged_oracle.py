"""Plain 64-bit implementations of the page-scaled cache's operators and of the logits' adjustment (any device)."""
import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def page_scale(amax: float, qmax: float) -> float:
    """The smallest power of two s >= 2^-126 with amax <= qmax * s."""
    s = 2.0 ** -126
    while s * qmax < amax:
        s *= 2.0
    return s


def encode(x: torch.Tensor, dtype) -> torch.Tensor:
    """float64 values (already divided by the scale) -> the codes' values, round to nearest even; NaN -> 0."""
    q = QMAX[dtype]
    x = torch.nan_to_num(x, nan=0.0, posinf=q, neginf=-q).clamp(-q, q)
    if dtype == torch.int8:
        return torch.round(x)
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e): 3 fraction bits, and 2^-9 at least
    unit = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / unit) * unit


class PageCache:
    """The values that a cache's codes stand for before scaling, and its scales, in 64 bits; keys or values of one layer."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, page: int):
        self.dtype, self.page = codes.dtype, page
        self.codes, self.scale = codes.double().clone(), scale.double().clone()

    def append(self, rows: torch.Tensor, slots) -> None:
        """rows [T, Hkv, Dh] in the order of the slots, one run of a page after another."""
        rows = rows.double()
        t = 0
        while t < len(slots):
            e = t + 1
            while e < len(slots) and slots[e] == slots[e - 1] + 1 and slots[e] % self.page:
                e += 1
            if slots[t] >= 0:
                self._run(rows[t:e], slots[t])
            t = e

    def _run(self, rows, slot):
        pg, first = divmod(slot, self.page)
        for h in range(rows.shape[1]):
            x = rows[:, h]
            fine = x[torch.isfinite(x)].abs()
            now = page_scale(float(fine.max()) if fine.numel() else 0.0, QMAX[self.dtype])
            if first:
                old = float(self.scale[pg, h])
                now = max(now, old)
                held = self.codes[pg * self.page:slot, h]
                self.codes[pg * self.page:slot, h] = encode(held * (old / now), self.dtype)
            self.codes[slot:slot + len(rows), h] = encode(x / now, self.dtype)
            self.scale[pg, h] = now

    def values(self, slots: torch.Tensor) -> torch.Tensor:
        return self.codes[slots] * self.scale[slots // self.page][:, :, None]


def attention(q, k, v, ctx, q_len, scale=None):
    """q [q_len, Hq, Dh], k / v [ctx, Hkv, Dh] (float64) -> (out, sum of p |v|), both [q_len, Hq, Dh]."""
    hq, dh = q.shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    for j in range(q_len):
        n = ctx - q_len + j + 1
        if n <= 0:
            continue
        kj = k[:n].repeat_interleave(hq // k.shape[1], dim=1)
        vj = v[:n].repeat_interleave(hq // k.shape[1], dim=1)
        p = torch.softmax(torch.einsum("hd,thd->ht", q[j], kj) * scale, dim=-1)
        out[j] = torch.einsum("ht,thd->hd", p, vj)
        mag[j] = torch.einsum("ht,thd->hd", p, vj.abs())
    return out, mag


def token_counts(prompt, output, vocab):
    """int64 [vocab] in the table's packing (bit 15 = in the prompt), as int16 values."""
    c = [0] * vocab
    for t in output:
        c[t] = min(c[t] + 1, 32767)
    for t in set(prompt):
        c[t] -= 32768
    return torch.tensor(c)


def adjust(z, counts, penalties, bias, allowed):
    """One row: z [V] float64, counts [V] (packed) or None, penalties (r, f, p), bias {id: b}, allowed bool [V] or None."""
    z = z.clone()
    if counts is not None:
        r, f, p = penalties
        made = counts & 0x7FFF
        z = torch.where(counts != 0, torch.where(z > 0, z / r, z * r), z)
        z = z - torch.where(made > 0, f * made + p, torch.zeros_like(z))
    for i, b in (bias or {}).items():
        z[i] += b
    if allowed is not None:
        z[~allowed] = -math.inf
    return z
