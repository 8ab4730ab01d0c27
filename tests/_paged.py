"""Plain 64-bit statements of the paged-cache operators, and caches to try them on (CPU)."""
import torch

F64 = torch.float64
U_BF16, U_F32 = 2.0 ** -8, 2.0 ** -24          # one rounding, relative


def make_cache(lens, hk, hd, page, g, spare=2, poison=True, cols=None):
    """pages in random order; rows that belong to no token hold NaN. -> k, v [pages, hk, page, hd] bf16, table int32 [B, cols]"""
    need = [-(-n // page) for n in lens]
    cols = max(1, max(need)) if cols is None else cols
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    k = torch.randn(pages, hk, page, hd, generator=g).bfloat16()
    v = torch.randn(pages, hk, page, hd, generator=g).bfloat16()
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        for j in range(0, n, page):
            used[int(table[b, j // page]), :min(page, n - j)] = True
    if poison:
        k.masked_fill_(~used[:, None, :, None], float('nan'))
        v.masked_fill_(~used[:, None, :, None], float('nan'))
    return k, v, table


def tokens(pages, table, b, n, hk):
    """rows of head hk of the first n tokens of sample b in order, fp64, and which of them are there"""
    page = pages.shape[2]
    j = torch.arange(n)
    pg = table[b].long()[j // page]
    ok = (pg >= 0) & (pg < pages.shape[0])
    x = pages[pg.clamp(0, pages.shape[0] - 1), hk, j % page].to(F64)
    return torch.where(ok[:, None], x, torch.zeros((), dtype=F64)), ok


def attention(q, k, v, table, new, lens, scale, row_of_pos=None, weights=None):
    """-> out, its tolerance, lse, its tolerance, (weights, their tolerance): fp64. Tolerances from the roundings: a score is an hd-term
    fp32 sum, a probability is rounded to bf16 before P V, the result once more"""
    rows, hd = q.shape[0], k.shape[3]
    hkn = k.shape[1]
    H = q.shape[1] // hd
    G = H // hkn
    out, tol = torch.zeros(rows, H * hd, dtype=F64), torch.zeros(rows, H * hd, dtype=F64)
    lse, ltol = torch.zeros(H, rows, dtype=F64), torch.zeros(H, rows, dtype=F64)
    w = weights.to(F64).clone() if weights is not None else None
    wtol = w.abs() * 2 * U_F32 if w is not None else None
    p0 = 0
    for b, (n, L) in enumerate(zip(new, lens)):
        pos = torch.arange(p0, p0 + n)
        r = row_of_pos.long()[pos] if row_of_pos is not None else pos
        for h in range(H):
            kk, ok = tokens(k, table, b, L, h // G)
            vv, _ = tokens(v, table, b, L, h // G)
            qq = q[r, h * hd:(h + 1) * hd].to(F64)
            seen = (torch.arange(L)[None] <= (L - n + torch.arange(n))[:, None]) & ok[None]
            s = torch.where(seen, qq @ kk.T * scale, float('-inf'))
            ds = (qq.abs() @ kk.abs().T * scale * (hd + 4) * U_F32)            # hd products summed in fp32, scaled
            ds = torch.where(seen, ds, 0.0).amax(1) if L else torch.zeros(n, dtype=F64)
            z = torch.logsumexp(s, 1) if L else torch.full((n,), float('-inf'), dtype=F64)
            p = torch.where(seen, torch.exp(s - torch.where(z.isinf(), 0.0, z)[:, None]), 0.0)
            o, a = p @ vv, p @ vv.abs()
            rel = 2 * ds + (L + 64) * U_F32                                    # numerator and denominator of a probability
            out[r, h * hd:(h + 1) * hd] = o
            # rounding of the probabilities, the fp32 sum over the tokens, rounding of the result (which acts on what the others left)
            e = a * (U_BF16 + rel[:, None] + (L + 8) * U_F32)
            tol[r, h * hd:(h + 1) * hd] = e + (o.abs() + e) * U_BF16
            lse[h, pos] = z
            zt = ds + (L + 64) * U_F32 + 8 * U_F32 * torch.where(z.isinf(), 0.0, z).abs()
            ltol[h, pos] = zt
            if w is not None:
                w[b, h // G, :L] += p.sum(0)
                wtol[b, h // G, :L] += (p * (ds + zt + 16 * U_F32 + (G * n + 2) * U_F32)[:, None]).sum(0) + p.sum(0) * 2 * U_F32
        p0 += n
    return (out, tol, lse, ltol) if w is None else (out, tol, lse, ltol, w, wtol)


def append(qkv, row_seq, row_index, table, k, v, row_pos, cos, sin, H):
    """-> q, its tolerance, k, its tolerance, v (k / v: the whole pools)"""
    pages, hk, page, hd = k.shape
    half = hd // 2
    x = qkv.view(-1, H + 2 * hk, hd).to(F64)
    pos = row_pos.long().clamp(0, cos.shape[0] - 1)
    c, s = cos[pos].to(F64)[:, None], sin[pos].to(F64)[:, None]
    lo, hi = x[..., :half], x[..., half:]
    y = torch.cat([lo * c[..., :half] - hi * s[..., :half], hi * c[..., half:] + lo * s[..., half:]], -1)
    mag = torch.cat([(lo * c[..., :half]).abs() + (hi * s[..., :half]).abs(), (hi * c[..., half:]).abs() + (lo * s[..., half:]).abs()], -1)
    tol = y.abs() * U_BF16 + mag * 4 * U_F32 * (1 + U_BF16)
    kk, vv, kt = k.to(F64), v.to(F64), torch.zeros(k.shape, dtype=F64)
    for r in range(x.shape[0]):
        b, j = int(row_seq[r]), int(row_index[r])
        if not (0 <= b < table.shape[0]) or not (0 <= j < table.shape[1] * page):
            continue
        pg = int(table[b, j // page])
        if not 0 <= pg < pages:
            continue
        kk[pg, :, j % page], kt[pg, :, j % page] = y[r, H:H + hk], tol[r, H:H + hk]
        vv[pg, :, j % page] = x[r, H + hk:]
    return y[:, :H].reshape(-1, H * hd), tol[:, :H].reshape(-1, H * hd), kk, kt, vv


def evict(weights, table, n_pages, page, lens, budget, recent):
    """-> kept: list [B][hk] of index lists, new lens"""
    kept, new = [], []
    for b, L in enumerate(lens):
        L = max(0, min(L, table.shape[1] * page, weights.shape[2]))
        there = [j for j in range(L) if 0 <= int(table[b, j // page]) < n_pages]
        n = min(len(there), budget)
        row = []
        for h in range(weights.shape[1]):
            ws = weights[b, h].tolist()
            key = lambda j: (0 if j >= L - min(recent, L) else 1, 0.0 if j >= L - min(recent, L) else (float('inf') if ws[j] != ws[j] else -ws[j]),  # noqa: E731
                             0 if j >= L - min(recent, L) or ws[j] == ws[j] else 1, j)
            row.append(sorted(sorted(there, key=key)[:n]))
        kept.append(row)
        new.append(n)
    return kept, new
