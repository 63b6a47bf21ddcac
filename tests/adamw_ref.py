"""AdamW with 8-bit states, written down in 64 bits on the CPU for the tests (one tensor at a time, numbers looked up in a list)."""
import math

import torch

BLOCK = 256


def numbers(signed):
    """Every finite number >= 0 of the form, in the order of its codes 0, 1, 2, ...: e4m3 (to 448) or e5m3 without a sign (to 61440)."""
    low, top = (-6, 448.0) if signed else (-14, 61440.0)
    got = [i * 2.0 ** (low - 3) for i in range(8)]
    e = low
    while 2.0 ** e <= top:
        got += [2.0 ** e * (1 + i / 8) for i in range(8) if 2.0 ** e * (1 + i / 8) <= top]
        e += 1
    return torch.tensor(got, dtype=torch.float64)


def four_bits(a):
    """a >= 0 to four significant bits, to nearest, ties to even."""
    mant, e = torch.frexp(a)
    return torch.ldexp(torch.round(mant * 16), e - 4)


def scale_of(block, signed):
    """The power of two of a block (its finite magnitudes below 2^128 count)."""
    a = block.abs()
    a = torch.where(torch.isfinite(a), four_bits(torch.where(torch.isfinite(a), a, torch.zeros_like(a))), torch.zeros_like(a))
    a = a[a < 2.0 ** 128]
    top, largest = (a.max().item() if a.numel() else 0.0), 448.0 if signed else 61440.0
    k = -126 if top == 0 else max(-126, math.frexp(top)[1] - 30)
    while top > largest * 2.0 ** k:
        k += 1
    return k


def hold(x, signed):
    """x (1-D, f64) as the 8-bit form holds it; and the blocks' exponents."""
    out, ks, table = torch.empty_like(x), [], numbers(signed)
    mid = (table[1:] + table[:-1]) / 2
    for b in range(0, x.numel(), BLOCK):
        blk = x[b:b + BLOCK]
        k = scale_of(blk, signed)
        a = blk.abs() * 2.0 ** -k
        code = torch.bucketize(a, mid)                                       # the lower one on a tie ...
        tie = (code < mid.numel()) & (a == mid[code.clamp_max(mid.numel() - 1)])
        code = code + (tie & (code % 2 == 1)).long()                         # ... unless the higher one is even
        if not signed:
            code = torch.where((blk > 0) & (code == 0), torch.ones_like(code), code)
        y = table[code.clamp_max(table.numel() - 1)] * 2.0 ** k * torch.sign(blk)
        over = ~torch.isfinite(blk) | (four_bits(torch.where(torch.isfinite(blk), blk.abs(), torch.zeros_like(blk))) >= 2.0 ** 128)
        y = torch.where(over, torch.full_like(y, math.nan) if signed else torch.where(torch.isnan(blk), blk, torch.full_like(blk, math.inf)), y)
        out[b:b + BLOCK] = y
        ks.append(k)
    return out, ks


def clip_of(gs, max_norm):
    """(norm, coefficient) over a list of gradients."""
    norm = math.sqrt(sum(float((g.double().cpu().flatten() ** 2).sum()) for g in gs))
    return norm, min(1.0, max_norm / (norm + 1e-6)) if not math.isnan(norm) else math.nan


def step(p, g, m, v, t, lr, betas, eps, wd, c=1.0):
    """One update of one tensor (1-D, f64; t = number of this step): (p', m', v', and scales for tolerances: |update| with sums taken by
    magnitude, |b1 m| + |a1 g|)."""
    b1, b2 = betas
    g = g * c
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = torch.sqrt(v2) / math.sqrt(1 - b2 ** t) + eps
    step_size = lr / (1 - b1 ** t)
    mag = (b1 * m).abs() + ((1 - b1) * g).abs()
    return p * (1 - lr * wd) - step_size * m2 / den, m2, v2, step_size * mag / den, mag
