"""Plain 64-bit statements of the paged-cache operators and of sampling, used
by their GPU tests: loops over sequences, heads and rows, nothing shared with
the kernels."""

from __future__ import annotations

import math

import torch

# half of the spacing of the numbers next to 1: the relative error of one rounding
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make_cache(lens, kv_heads, page, d, dtype, device, seed, junk=float("nan"), width=None):
    """Pages in shuffled order whose unused slots hold ``junk``, the table (-1 where unused), and each
    sequence's keys and values [kv_heads, n, d] in 64 bits."""

    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    num = sum(need) + 3
    order = torch.randperm(num, generator=g).tolist()
    k = torch.full((num, kv_heads, page, d), junk, dtype=dtype)
    v = torch.full((num, kv_heads, page, d), junk, dtype=dtype)
    table = torch.full((max(len(lens), 1), width or max(need + [1])), -1, dtype=torch.int32)
    keys, vals, at = [], [], 0
    for b, n in enumerate(lens):
        kk = torch.randn((kv_heads, n, d), generator=g).to(dtype)
        vv = torch.randn((kv_heads, n, d), generator=g).to(dtype)
        for j in range(need[b]):
            table[b, j] = order[at]
            m = min(page, n - j * page)
            k[order[at], :, :m] = kk[:, j * page:j * page + m]
            v[order[at], :, :m] = vv[:, j * page:j * page + m]
            at += 1
        keys.append(kk.double())
        vals.append(vv.double())
    return k.to(device), v.to(device), table[:len(lens)].to(device), keys, vals


def starts(new, device):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device)


def attention(q, new, lens, keys, vals, scale):
    """(out, lse, sum_j p_j |v_j|, the largest sum |q k| scale of the row's keys), 64 bits, on the CPU."""

    rows, heads, d = q.shape
    out = torch.zeros((rows, heads, d), dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros((rows, heads), dtype=torch.float64)
    q = q.double()
    at = 0
    for b, (t, n) in enumerate(zip(new, lens)):
        group = heads // keys[b].shape[0] if len(keys) else 1
        for i in range(t):
            count = n - t + i + 1
            if count > 0:
                for h in range(heads):
                    kk, vv = keys[b][h // group, :count], vals[b][h // group, :count]
                    s = kk @ q[at + i, h] * scale
                    p = torch.softmax(s, 0)
                    out[at + i, h] = p @ vv
                    mag[at + i, h] = p @ vv.abs()
                    lse[at + i, h] = torch.logsumexp(s, 0)
                    reach[at + i, h] = (kk.abs() @ q[at + i, h].abs()).max() * scale
        at += t
    return out, lse, mag, reach


def sample_row(x, t, k, p, low, u):
    """(token, log-probability) of one row by the definition, masses in 64 bits."""

    x = [-math.inf if math.isnan(v) else v for v in x]
    m = max(x)
    if m == -math.inf:
        return -1, -math.inf
    if not t > 0:
        return x.index(m), 0.0
    w = [1.0 if v == m else math.exp((v - m) / t) if v > -math.inf and m < math.inf else 0.0 for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        total, run, kept = sum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and run >= p * total:
                break
            kept.append(i)
            run += w[i]
        order = kept
    kept = sorted(i for i in order if w[i] >= min(low, 1.0))
    whole, run = sum(w[i] for i in kept), 0.0
    for i in kept:
        run += w[i]
        if run > u * whole:
            return i, math.log(w[i] / whole)
    return kept[-1], math.log(w[kept[-1]] / whole)
