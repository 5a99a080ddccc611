"""Plain forms of the 8-bit cache's operators and of the verification of drafts, row by row, for the tests.

The write is restated in 32 bits, operation by operation (each product, sum and difference is one rounding, so the
kernel's bytes have to be the same); everything else is in 64 bits."""

import math

import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def power(byte):
    """2^(byte - 127) in 64 bits."""
    return (byte.long() - 127 + 1023 << 52).view(torch.float64)


def scale_byte(amax):
    """The smallest byte of 1 and more with amax <= 448 * 2^(byte - 127): by trying them, from the definition."""
    out = torch.ones(amax.shape, dtype=torch.int64)
    for b in range(253, 0, -1):
        out = torch.where(amax.double() <= 448.0 * 2.0 ** (b - 127), torch.full_like(out, b), out)
    return out


def round_e4m3(x):
    """64-bit x (|x| <= 448 or no number) to e4m3, to nearest with ties to even."""
    _, e = torch.frexp(x)
    step = 2.0 ** ((e - 1).clamp(min=-6) - 3).double()
    return torch.where(x.isfinite(), torch.round(x / step) * step, math.nan).to(torch.float32).to(E4M3)


def rotate32(x, cos, sin, positions, interleaved):
    """x float32 [n, heads, hd]; products and differences rounded one by one."""
    if cos is None:
        return x.clone()
    half = cos.shape[1]
    i0 = torch.arange(half) * (2 if interleaved else 1)
    i1 = i0 + 1 if interleaved else i0 + half
    c, s = cos[positions][:, None], sin[positions][:, None]
    out = x.clone()
    out[..., i0] = x[..., i0] * c - x[..., i1] * s
    out[..., i1] = x[..., i0] * s + x[..., i1] * c
    return out


def write(qkv, rows, cos, sin, pages, scales, table, page_size, H, G, hd, interleaved, do_write=True, bias=None):
    """rows: [(positions before, new tokens)].  Changes pages / scales (uint8 views) in place; returns q [n, H * hd] in
    qkv's dtype (rows behind the last row: None of them is looked at)."""
    block = page_size // scales.shape[3]
    n = sum(m for _, m in rows)
    x = qkv[:n].float()
    if bias is not None:
        x = x + bias
    x = x.view(n, H + 2 * G, hd)
    positions = torch.tensor([b + i for b, m in rows for i in range(m)], dtype=torch.long)
    qk = rotate32(x[:, :H + G], cos, sin, positions, interleaved)
    kv = torch.stack([qk[:, H:], x[:, H + G:]], 1)                   # [n, 2, G, hd]
    at = 0
    for r, (before, m) in enumerate(rows):
        for b0 in range(before // block * block, before + m, block) if do_write and m else ():
            lo, hi = max(before, b0), min(before + m, b0 + block)
            new = kv[at + lo - before:at + hi - before]              # [t, 2, G, hd]
            byte = scale_byte(torch.where(new.isfinite(), new.abs(), torch.zeros(())).amax((0, 3)))
            page, cell = int(table[r, b0 // page_size]), b0 % page_size
            held = pages[page, :, :, cell:cell + lo - b0]            # [2, G, old, hd]
            if lo > b0:
                had = scales[page, :, :, cell // block].long()
                grown = torch.maximum(byte, had)
                again = round_e4m3(held.contiguous().view(E4M3).double() * (power(had) / power(grown))[..., None, None])
                held.copy_(again.view(torch.uint8))
                byte = grown
            scales[page, :, :, cell // block] = byte.to(torch.uint8)
            value = round_e4m3(new.double() / power(byte)[None, :, :, None])
            pages[page, :, :, cell + lo - b0:cell + hi - b0] = value.view(torch.uint8).permute(1, 2, 0, 3)
        at += m
    return qk[:, :H].reshape(n, -1).to(qkv.dtype)


def values(pages, scales, table_row, length, page_size):
    """Keys and values in 64 bits, [2, length, G, hd], of a row's first tokens."""
    block = page_size // scales.shape[3]
    ids = table_row[:-(-length // page_size)].long()
    x = pages[ids].view(E4M3).double().unflatten(3, (page_size // block, block)) * power(scales[ids])[..., None, None]
    return x.flatten(3, 4).permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :length]


def attend(q, pages, scales, table, rows, page_size, H, G, hd, scale, window=0):
    """(out [n, H * hd], spread [n, H * hd], reach [n, H, 1]): spread is sum_j p_j |v_j|, reach the largest scale * sum |q k|
    among the keys that a query sees, for the tolerance."""
    out, spread, reach, at = [], [], [], 0
    for r, (before, m) in enumerate(rows):
        if m == 0:
            continue
        k, v = values(pages, scales, table[r], before + m, page_size)
        k, v = k.repeat_interleave(H // G, 1), v.repeat_interleave(H // G, 1)
        x = q[at:at + m].double().view(m, H, hd)
        far = torch.arange(before, before + m)[:, None] - torch.arange(before + m)
        seen = (far >= 0) & (far < (window or before + m + 1))
        for i in range(m):                                            # (only keys that are seen: NaN stays with them)
            ks, vs = k[seen[i]], v[seen[i]]
            s = torch.einsum("hd,khd->hk", x[i], ks) * scale
            p = torch.softmax(s, -1)
            out.append(torch.einsum("hk,khd->hd", p, vs))
            spread.append(torch.einsum("hk,khd->hd", p, vs.abs()))
            reach.append((torch.einsum("hd,khd->hk", x[i].abs(), ks.abs()) * abs(scale)).amax(-1, keepdim=True))
        at += m
    return torch.stack(out).view(-1, H * hd), torch.stack(spread).view(-1, H * hd), torch.stack(reach)


def verify(probs, drafts, counts, uniforms, draft_probs=None):
    """(tokens, accepted) as lists, in 64 bits, draft by draft."""
    tokens, accepted, d0 = [], [], 0
    p, u = probs.double(), uniforms.double().tolist()
    for r, k in enumerate(counts):
        at, x = d0 + r, drafts[d0:d0 + k].tolist()
        i = 0
        while i < k and 0 <= x[i] < p.shape[1] and \
                u[at + i] * (1.0 if draft_probs is None else float(draft_probs[d0 + i, x[i]])) < float(p[at + i, x[i]]):
            i += 1
        full = torch.nan_to_num(p[at + i], nan=0.0).clamp(min=0.0)
        w = full.clone()
        if i < k and draft_probs is None:
            if 0 <= x[i] < len(w):
                w[x[i]] = 0.0
        elif i < k:
            w = torch.nan_to_num(p[at + i] - draft_probs[d0 + i].double(), nan=0.0).clamp(min=0.0)
        if float(w.sum()) <= 0.0:
            w = full
        total = torch.cumsum(w, 0)
        token = -1
        if float(total[-1]) > 0.0:
            past = (total > u[at + k] * float(total[-1])).nonzero()
            token = int(past[0]) if len(past) else int((w > 0).nonzero()[-1])
        tokens += x[:i] + [token] + [-1] * (k - i)
        accepted.append(i)
        d0 += k
    return tokens, accepted
