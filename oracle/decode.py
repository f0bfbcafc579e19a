"""The autoregressive-decoding operators in 64 bits, from their formulas (test infrastructure; CPU, loops over sequences and heads)."""
import math

import torch


def turned(x, positions, freq, amplitude=1.0, interleaved=False):
    """x [tokens, heads, dim] with pair i of every head turned by positions[t] * freq[i] (radians)."""
    out, rd = x.double().clone(), 2 * len(freq)
    a = positions.double()[:, None] * torch.as_tensor(freq, dtype=torch.float64)
    c, s = (amplitude * torch.cos(a))[:, None], (amplitude * torch.sin(a))[:, None]
    one, two = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    x1, x2 = x.double()[..., one], x.double()[..., two]
    out[..., one], out[..., two] = x1 * c - x2 * s, x2 * c + x1 * s
    return out


def places(table, seq_lens, q_starts, page_size, pages, tokens):
    """Per sequence: its new tokens, their positions, and for every key position the (page, row) that holds it, or None."""
    out = []
    for b, length in enumerate(seq_lens):
        start = min(max(q_starts[b], 0), tokens)
        n = min(max(q_starts[b + 1], start), tokens) - start
        length = max(length, 0)
        where = []
        for p in range(length):
            col = p // page_size
            page = table[b][col] if col < len(table[b]) else -1
            where.append((page, p % page_size) if 0 <= page < pages else None)
        out.append((start, n, [length - n + i for i in range(n)], where))
    return out


def attend(q, k_cache, v_cache, table, seq_lens, q_starts, scale, causal=True, window=0):
    """-> out [tokens, heads, dim] (NaN in rows no sequence owns), the sum of p |v| per value, and the largest sum of |q k scale|."""
    tokens, heads, dim = q.shape
    pages, kv_heads, page_size, _ = k_cache.shape
    g = heads // kv_heads
    out = torch.full((tokens, heads, dim), math.nan, dtype=torch.float64)
    mag, reach = torch.zeros_like(out), 0.0
    for start, n, pos, where in places(table, seq_lens, q_starts, page_size, pages, tokens):
        keys = [j for j, w in enumerate(where) if w is not None]
        if n == 0:
            continue
        out[start: start + n] = 0
        if not keys:
            continue
        at = torch.tensor([where[j] for j in keys])
        k, v = (c[at[:, 0], :, at[:, 1]].double() for c in (k_cache, v_cache))           # [keys, kv_heads, dim]
        gap = torch.tensor(pos)[:, None] - torch.tensor(keys)[None]
        seen = torch.ones_like(gap, dtype=torch.bool)
        if causal:
            seen &= gap >= 0
        if window:
            seen &= gap < window
        for h in range(heads):
            kh, vh, qh = k[:, h // g], v[:, h // g], q[start: start + n, h].double()
            s = torch.where(seen, qh @ kh.T * scale, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
            l = p.sum(-1, keepdim=True)
            p = torch.where(l > 0, p / l, 0.0)
            for i in range(n):          # a key that is not seen takes no part, whatever it holds
                row = seen[i]
                out[start + i, h] = p[i, row] @ vh[row]
                mag[start + i, h] = p[i, row] @ vh[row].abs()
                if bool(row.any()):
                    reach = max(reach, float((qh[i].abs() @ kh[row].abs().T).max()) * abs(scale))     # a score is off by its size, whatever its sign
    return out, mag, reach


def linear_w4(x, qweight, scales, zeros=None, bias=None):
    """-> y [m, n] and the sum of |x w| per value."""
    n, half = qweight.shape
    levels = torch.zeros(n, 2 * half, dtype=torch.float64)
    levels[:, 0::2], levels[:, 1::2] = (qweight & 15).double(), (qweight >> 4).double()
    group = 2 * half // scales.shape[1]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)
    w = (levels - z) * scales.double().repeat_interleave(group, 1)
    y = x.double() @ w.T
    return (y if bias is None else y + bias.double()), x.double().abs() @ w.abs().T
