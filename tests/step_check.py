"""A packed step's attention operators from their definitions in 64 bits, on the CPU: how rows lie, what the cache
keeps, norms and rotation, attention, and the bounds that each result has to keep."""
import math

import torch

HALF = 2.0 ** -8      # half a step of bf16, relative
LEAST = 2.0 ** -100   # the least scale of a kept vector
F32 = 2.0 ** -24


def packed(runs, lengths, page, seed=0, spare=2, shared=0, pad=0):
    """(starts, lengths, table, pages): pages in no order, the first `shared` tokens' the same for all requests, -1 behind
    the last ones. `pad`: columns of the table's buffer that are not its own."""
    gen = torch.Generator().manual_seed(seed)
    common = shared // page
    need = [max(0, -(-n // page) - common) for n in lengths]
    pages = common + sum(need) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    wide = torch.full((len(runs), common + max(need + [1]) + pad), -1, dtype=torch.int32)
    at = common
    for r, n in enumerate(need):
        wide[r, :common] = order[:common]
        wide[r, common : common + n] = order[at : at + n]
        at += n
    starts = torch.tensor([sum(runs[:r]) for r in range(len(runs) + 1)], dtype=torch.int32)
    return starts, torch.tensor(lengths, dtype=torch.int32), wide[:, : wide.shape[1] - pad] if pad else wide, max(pages, 1)


def places(starts, lengths, table, page, pages, rows):
    """[(request, position, page or None, place)] of each row; None for a row of no request."""
    got = []
    for m in range(rows):
        r = max((i for i in range(len(starts)) if starts[i] <= m), default=-1)
        if r < 0 or r >= len(lengths):
            got.append(None)
            continue
        p = int(lengths[r]) - int(starts[r + 1]) + m
        column = p // page if p >= 0 else -1
        found = int(table[r, column]) if 0 <= column < table.shape[1] else -1
        got.append((r, p, found if 0 <= found < pages else None, p % page))
    return got


def rotated(x, weight, frequencies, positions, eps):
    """(y, bound): the norm and the rotation in 64 bits, and what fp32 and one rounding to bf16 may leave of it.

    fp32: the mean of squares is off by (dim / 16 + 5) 2^-24 at most (a lane adds dim / 16 squares, four additions across a
    vector's lanes), of which the root leaves half, and the root, the quotient and the products by six more: below (dim / 64 + 16) 2^-24
    in all; an angle's fraction, cosine and sine by 2^-22 of the pair."""
    y = x.double()
    dim = y.shape[-1]
    off = torch.zeros_like(y)
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))).sqrt() * weight.double()
        off = y.abs() * (dim / 64 + 16) * F32
    if frequencies is not None:
        h = frequencies.numel()
        angle = positions.double()[:, None, None] * frequencies.double()
        a, b = y[..., :h].clone(), y[..., h : 2 * h].clone()
        pair = (a.abs() + b.abs()) * (2.0 ** -22 + 4 * F32) + off[..., :h] + off[..., h : 2 * h]
        y, off = y.clone(), off.clone()
        y[..., :h], y[..., h : 2 * h] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
        off[..., :h] = off[..., h : 2 * h] = pair
    return y, off


def check_bf16(got, want, off, label=""):
    """got (bf16) is a rounding of something within `off` of want."""
    bound = want.abs() * HALF + off * (1 + HALF) + 2.0 ** -133
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), f"{label}: off by up to {float((d / bound).max())} of the bound"


def kept(x):
    """(codes, scales) of vectors along the last dimension, as the cache keeps them."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    most = torch.where(bad, 1.0, x.abs().amax(-1, keepdim=True))
    small = most / 127 < LEAST
    codes = torch.where(small, x / LEAST, x * 127 / torch.where(small, 1.0, most)).round()
    scales = torch.where(small, LEAST, most / 127)
    return torch.where(bad, 0.0, codes), torch.where(bad, math.nan, scales.float().double())


def attended(q, k, v, position, scale):
    """(out, bound) of one request: q [n, heads, dim] bf16, k and v [tokens, kv heads, dim] in 64 bits as the cache's values,
    row i at position[i]; a key that is None (NaN-free mask `hidden`) has weight 0.

    The bound: weights in fp16 (2^-11 of each, below 2^-14 of the row's largest weight times scale half a step of 2^-24), their
    exponents from fp32 sums of dim products (2^-24 of the products' size for each, twelve more for what follows)
    and one rounding to bf16 (check_bf16 adds it)."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out, off = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dim, dtype=torch.float64)
    hidden = torch.arange(k.shape[0])[None, :] > position[:, None]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h].double() @ kh.T * scale).masked_fill(hidden, -math.inf)
        size = (q[:, h].double().abs() @ kh.abs().T * scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        seen = ~hidden.all(1)
        w = torch.zeros_like(s)
        w[seen] = torch.softmax(s[seen], 1)
        out[:, h] = w @ vh
        exponent = size * F32 * (dim / 8 + 12) + 64 * F32
        largest = (w * vh.abs().amax(1)).amax(1, keepdim=True)
        off[:, h] = (w @ vh.abs()) * (2.0 ** -11 + 2 * exponent) + out[:, h].abs() * 2 * exponent + largest * 2.0 ** -24 * (~hidden).sum(1, keepdim=True)
    return out, off
