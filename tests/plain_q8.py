"""Plain 64-bit forms of the 8-bit cache's operators and of the verification of drafted tokens, written
from their definitions; sequence by sequence, in numpy and torch on the CPU."""
import math

import numpy as np
import torch

PAGE = 64
LIMIT = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
FORMATS = [torch.float8_e4m3fn, torch.int8]


def quantise(x, fmt):
    """Codes and float32 scales of float32 vectors, in the operations and types of the definition."""
    limit = LIMIT[fmt]
    bad = ~torch.isfinite(x).all(-1)
    a = torch.where(bad, torch.ones(()), x.abs().amax(-1)).clamp_min(2.0 ** -100)
    y = torch.where(bad.unsqueeze(-1), torch.zeros(()), x) * (torch.tensor(limit) / a).unsqueeze(-1)
    y = y.clamp(-limit, limit)
    code = y.to(fmt) if fmt == torch.float8_e4m3fn else y.round().to(torch.int8)
    return code, torch.where(bad, torch.tensor(float("nan")), a / torch.tensor(limit))


def values(code, scale):
    """What codes and scales stand for, in 64 bits."""
    return code.float().double() * scale.double().unsqueeze(-1)


def half_step(x, scale, fmt):
    """The most a rounding to the format may be off at the value x (both float64)."""
    if fmt == torch.int8:
        return scale.unsqueeze(-1).expand_as(x) / 2
    return torch.maximum(x.abs() * 2.0 ** -4, scale.unsqueeze(-1) * 2.0 ** -10)


def row_vectors(codes, scales, table, end, ring):
    """[positions, kv, dim] float64 of the positions ``first`` .. end - 1 that a row's pages hold, and first."""
    first = max(0, end - ring) if ring else 0
    out = []
    for p in range(first, end):
        place = p % ring if ring else p
        page = int(table[place // PAGE])
        out.append(values(codes[page, :, place % PAGE], scales[page, :, place % PAGE]))
    if not out:
        return torch.zeros((0, codes.shape[1], codes.shape[3]), dtype=torch.float64), first
    return torch.stack(out), first


def attention(q, pages, cu, ends, table, ring, n_heads, n_kv, window, scale):
    """(output, sum_j p_j |v_j|, the largest p_j vs_j, the largest scale * sum_d |q_d k_jd|, keys seen), float64."""
    k8, v8, ks, vs = (t.cpu() for t in pages)
    q = q.double().cpu()
    out = torch.zeros_like(q)
    mass, top, size = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    keys = torch.zeros(q.shape[0], dtype=torch.float64)
    for b, end in enumerate(ends):
        k, first = row_vectors(k8, ks, table[b], end, ring)
        v, _ = row_vectors(v8, vs, table[b], end, ring)
        vscale, _ = row_vectors(torch.ones_like(v8[..., :1], dtype=torch.float32), vs, table[b], end, ring)
        count = cu[b + 1] - cu[b]
        for i in range(count):
            t, pos = cu[b] + i, end - count + i
            lo = max(first, pos - window + 1 if window else 0)
            if pos + 1 <= lo:
                continue
            keys[t] = pos + 1 - lo
            for h in range(n_heads):
                hk = h // (n_heads // n_kv)
                kk, vv = k[lo - first:pos + 1 - first, hk], v[lo - first:pos + 1 - first, hk]
                s = (kk * q[t, h]).sum(-1) * scale
                p = torch.exp(s - s.max())
                p = p / p.sum()
                out[t, h] = (p.unsqueeze(-1) * vv).sum(0)
                mass[t, h] = (p.unsqueeze(-1) * vv.abs()).sum(0)
                top[t, h] = (p * vscale[lo - first:pos + 1 - first, hk, 0]).max()
                size[t, h] = ((kk * q[t, h]).abs().sum(-1)).max() * abs(scale)
    return out, mass, top, size, keys


def attention_tolerance(want, mass, top, size, keys, dtype, dim, fmt):
    """How far a kernel's output may be off, from its roundings.

    float32: a score is a sum of ``dim`` products, off by (dim + 8) 2^-24 of the sum of their magnitudes, and so is
    the exponential's argument; the exponential is off by 2 units in the last place and the sums over n keys
    by n + 8 roundings: relative to sum_j p_j |v_j|, twice (the sum of p as well).
    bfloat16 on the tensor cores: queries and codes are exact; a sum of products in the tensor cores may
    drop bits below 2^-22 of its largest term, a score times scales is rounded twice and a logarithm and
    two exponentials add 2^-21 at scores of the size of ``size``; weights are rounded to halves, 2^-11
    of each, 2^-25 of the largest below the normal range; the output is rounded once, 2^-8."""
    n = keys[:, None]
    if dtype == torch.float32:
        rel = 2 * ((dim + 8) * 2.0 ** -24 * (size + 1) + (n + 16) * 2.0 ** -24)
        return mass * rel[..., None] + want.abs() * 2.0 ** -24 + 1e-37
    if dim not in (64, 128):          # the generic kernel, rounded once
        rel = 2 * ((dim + 8) * 2.0 ** -24 * (size + 1) + (n + 16) * 2.0 ** -24)
        return mass * rel[..., None] + want.abs() * 2.0 ** -8 + 1e-37
    rel = 2.0 ** -11 + 2 * ((dim + 8) * 2.0 ** -22 * (size + 1) + 2.0 ** -20)
    small = 2.0 ** -25 * n * top * LIMIT[fmt]
    return mass * rel[..., None] + small[..., None] + want.abs() * 2.0 ** -8 + 1e-37


def halves_tolerance(want, mass, top, size, keys, most):
    """``attention_tolerance`` where keys and values are rounded to halves with their scales (2^-11 each): a score is off by
    2^-11 of the sum of its products' magnitudes and a probability relatively by twice that; probabilities are
    rounded to halves (2^-11), or by 2^-25 where the row's largest so far is 2^6 or more: 2^-31 of it, times a value
    of ``most`` at the largest, for each of n keys.  (A code of 2^-9 and a scale 2^-16 of the tile's largest are
    2^-20 of a half's range, rounded by 2^-25 at most: 2^-5 of the smallest code, which is 2^-23 of the vector's
    largest.)  The tensor cores' sums and the output as above."""
    n = keys[:, None]
    rel = 2 * (2.0 ** -11 + 2.0 ** -14) * size + 2 * 2.0 ** -11 + 2.0 ** -14 + 2.0 ** -18 * (size + 1)
    return mass * rel[..., None] + (2.0 ** -31 * n * most)[..., None] + want.abs() * 2.0 ** -8 + 1e-37


def softmax(row, temperature):
    d = row.astype(np.float64)
    if np.isnan(d).any() or np.isposinf(d).any() or not (d > -np.inf).any():
        return None
    e = np.exp((d - d.max()) / temperature)
    return e / e.sum()


def verify(logits, drafts, cu, draft_logits, accept_u, draw_u, temperature):
    """(accepted, tokens) of ``verify_drafts`` on numpy arrays."""
    accepted, tokens = [], []
    vocab = logits.shape[1]
    for b in range(len(draw_u)):
        n, row0 = cu[b + 1] - cu[b], cu[b] + b
        got, token = n, None
        for j in range(n + 1):
            row = logits[row0 + j]
            x = int(drafts[cu[b] + j]) if j < n else -2
            if temperature < 1e-6:
                best = -1 if np.isnan(row).any() or not (row > -np.inf).any() else int(np.argmax(row))
                if best < 0 or best != x:
                    got, token = j, best
                    break
                continue
            p = softmax(row, temperature)
            if p is None:
                got, token = j, -1
                break
            q = None
            if j < n:
                if draft_logits is not None:
                    q = softmax(draft_logits[cu[b] + j], temperature)
                if 0 <= x < vocab:
                    qx = 1.0 if draft_logits is None else (math.nan if q is None else q[x])
                    if float(accept_u[cu[b] + j]) * qx < p[x]:
                        continue
                left = p.copy()
                if draft_logits is None:
                    if 0 <= x < vocab:
                        left[x] = 0.0
                else:
                    left = np.zeros_like(p) if q is None else np.maximum(0.0, p - q)
                if left.sum() > 0:
                    p = left
            got = j
            sums = np.cumsum(p)
            above = np.nonzero((sums > float(draw_u[b]) * sums[-1]) & (p > 0))[0]
            token = int(above[0]) if above.size else int(np.nonzero(p > 0)[0][-1])
            break
        accepted.append(got)
        tokens.append(token)
    return accepted, tokens
