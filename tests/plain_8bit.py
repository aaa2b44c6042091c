"""What the operators over 8-bit weights and an 8-bit cache compute, step by step in 64 bits, with a bound of what rounding may add."""
from __future__ import annotations

import math

import torch

TOP, GROUP, PAGE = 448.0, 128, 64
PER_TOP = torch.tensor(1 / TOP, dtype=torch.float32)          # what the largest number is multiplied by for a scale


def as_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number in float64 (ties to even, beyond 448: 448; infinities and NaN: NaN)."""
    x = x.double()
    exponent = (torch.frexp(x)[1] - 1).clamp(min=-6)
    step = torch.exp2(exponent.double() - 3)
    y = ((x / step).round() * step).clamp(-TOP, TOP)
    return torch.where(torch.isfinite(x), y, math.nan)


def quantise_rows(x: torch.Tensor):
    """(values float64 [M, K], scales float32 [groups, M]): the scale and the division in float32, as they are defined."""
    m, k = x.shape
    x = x.float().cpu()
    groups = -(-k // GROUP)
    values, scales = torch.empty((m, k), dtype=torch.float64), torch.empty((groups, m))
    for g in range(groups):
        piece = x[:, g * GROUP:(g + 1) * GROUP]
        scales[g] = (piece.nan_to_num(0.0, math.inf, -math.inf).abs().amax(1) * PER_TOP).clamp(min=2.0 ** -100)
        values[:, g * GROUP:(g + 1) * GROUP] = as_e4m3(piece / scales[g][:, None])
    return values, scales


def quantise_weight(w: torch.Tensor):
    """(values float64 [N, K], scales float32 [row blocks, column blocks])."""
    n, k = w.shape
    w = w.float().cpu()
    values, scales = torch.empty((n, k), dtype=torch.float64), torch.empty((-(-n // GROUP), -(-k // GROUP)))
    for i in range(scales.shape[0]):
        for g in range(scales.shape[1]):
            at = (slice(i * GROUP, (i + 1) * GROUP), slice(g * GROUP, (g + 1) * GROUP))
            scales[i, g] = (w[at].abs().amax() * PER_TOP).clamp(min=2.0 ** -100)
            values[at] = as_e4m3(w[at] / scales[i, g])
    return values, scales


def product(x_values, x_scales, w_values, w_scales):
    """(y, bound): x W^T in float64, and what sums in float32 may be off by.  A group's 128 products are exact; each of its additions is off by at most one unit
    in the last place (tensor cores cut), 2^-23; a product of the scales, one with the sum and one addition a group: 2^-24 each."""
    x = x_values * x_scales.double().T.repeat_interleave(GROUP, 1)[:, :x_values.shape[1]]
    scale = w_scales.double().repeat_interleave(GROUP, 0)[:w_values.shape[0]].repeat_interleave(GROUP, 1)[:, :w_values.shape[1]]
    w = w_values * scale
    size = x.abs() @ w.abs().T
    return x @ w.T, size * (2 * GROUP + 2 + w_scales.shape[1]) * 2.0 ** -24


def power_for(largest: float) -> int:
    e = -40
    while e < 40 and TOP * 2.0 ** e < largest:
        e += 1
    return e


def treated(x, weight, eps, cos_sin, position, interleaved=False):
    """Heads [tokens, heads, d] normed (with a weight) and rotated (with a table)."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(2, keepdim=True) + eps).sqrt() * weight.double()
    if cos_sin is None:
        return x
    half = cos_sin.shape[1] // 2
    cos, sin = cos_sin.double()[position, None, :half], cos_sin.double()[position, None, half:]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    return y


def write(values, scales, rows, table, start, past):
    """Rows [tokens, heads, d] of one tensor (k or v) into pages values [pages, heads, 64, d] (float64, e4m3 numbers) and scales [pages, heads], in place: one
    sequence after the other, one page after the other."""
    for i in range(len(past)):
        for first in range(past[i], past[i] + start[i + 1] - start[i]):
            if first % PAGE and first != past[i]:
                continue
            last = min((first // PAGE + 1) * PAGE, past[i] + start[i + 1] - start[i])
            page, low = int(table[i, first // PAGE]), first % PAGE
            new = rows[start[i] + first - past[i]:start[i] + last - past[i]].double()
            for h in range(values.shape[1]):
                finite = new[:, h][torch.isfinite(new[:, h])].abs()
                power = power_for(float(finite.max()) if finite.numel() else 0.0)
                scale = max(float(scales[page, h]), 2.0 ** power) if low else 2.0 ** power
                if low:
                    values[page, h, :low] = as_e4m3(values[page, h, :low] * (float(scales[page, h]) / scale))
                values[page, h, low:low + last - first] = as_e4m3(new[:, h] / scale)
                scales[page, h] = scale


def attention(q, k, v, table, counts, past, scale, half_digits: int, split: bool = False):
    """(out, bound) for packed queries [tokens, heads, d] over held keys and values [pages, kv_heads, 64, d] (float64, scales within): ``counts`` queries of
    each sequence behind ``past`` earlier tokens.  The bound: a score's sum of d products off by 2^-23 of their sizes' sum each, its scaling and exponential by
    2^-21 of the score and 2^-21; a weight is rounded to ``half_digits`` binary digits; sums over the keys off by 2^-23 an addition, of which a block's
    order has at most 200 for a range of keys in turn and the joins, the others within an instruction.  ``split``: queries are the sum of two e4m3 numbers, the
    largest of a row between 2^7 and 2^8.  The nearest one leaves at most 2^-4 of an element, four binary digits of the eight of a bfloat16 number, which the second
    holds down to its last place, 2^-9: off by at most 2^-10, 2^-17 of the row's largest."""
    q = q.double().cpu()
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    at = 0
    for i, n in enumerate(counts):
        if past[i] + n > 0 and n > 0:
            total = past[i] + n
            pages = table[i, :-(-total // PAGE)].long()
            for h in range(heads):
                keys, values = (c[pages, h // group].reshape(-1, c.shape[3])[:total] for c in (k, v))
                rows = q[at:at + n, h]
                s = rows @ keys.T * scale
                off = (rows.abs() @ keys.abs().T * abs(scale)) * (keys.shape[1] + 4) * 2.0 ** -23 + s.abs() * 2.0 ** -21 + 2.0 ** -21
                if split:
                    off = off + rows.abs().amax(1, keepdim=True) * keys.abs().sum(1)[None, :] * abs(scale) * 2.0 ** -17
                hidden = torch.arange(total)[None, :] > past[i] + torch.arange(n)[:, None]
                p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1)
                off = off.masked_fill(hidden, 0.0).amax(1, keepdim=True)
                out[at:at + n, h] = p @ values
                bound[at:at + n, h] = (p @ values.abs()) * (2.0 ** -half_digits + 2 * off + (200 + total / 8) * 2.0 ** -23)
        at += n
    return out, bound
