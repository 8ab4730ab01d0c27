"""The paged cache of the generation path as four operators, for measurement: storing a chunk of new tokens (rotary positions
included), attention of the chunk over the cache, the attention weight every cached token has received, and eviction by it.

Layout (shared by both forms): `k_pages`, `v_pages` bf16 [pages, kv heads, page size, head dim]; `block_table` int32
[samples, pages per sample] names the pages of a sample in order; a sample's token j lies in page `block_table[b, j // size]`,
row `j % size`."""
import math

import torch

own = False

DEV = 'cuda'


# ---------------------------------------------------------------- cases
def listed():
    lm = dict(heads=32, kv_heads=32, dim=128, page=64)          # the decoder's own head layout
    return [
        # one decode step of eight conversations: the launch is what costs
        dict(name='append-decode-8', op='append', batch=8, new=1, kv=513, **lm),
        # prefill of four volumes at the longest prompt of the benchmark (4609 tokens): a pure copy rate
        dict(name='append-prefill-4x4609', op='append', batch=4, new=4609, kv=4609, **lm),
        # one token of one conversation right after a 2-D prompt: latency
        dict(name='decode-1x485', op='attn', batch=1, new=1, kv=485, **lm),
        # one token of eight conversations about volumes: the cache is read once
        dict(name='decode-8x4609', op='attn', batch=8, new=1, kv=4609, **lm),
        # a serving batch with grouped heads and long histories
        dict(name='decode-gqa-32x16384', op='attn', batch=32, new=1, kv=16384, heads=32, kv_heads=8, dim=128, page=128),
        # follow-up question of 37 tokens to a volume report, packed rows in expert order
        dict(name='chunk-4x37-of-2086', op='attn', batch=4, new=37, kv=2086, packed=True, **lm),
        # a long prompt taken in pieces: 512 new tokens over a long cache
        dict(name='chunk-1x512-of-8704', op='attn', batch=1, new=512, kv=8704, **lm),
        # the whole prompt of four volumes at once
        dict(name='prefill-4x4609', op='attn', batch=4, new=4609, kv=4609, packed=True, **lm),
        # decode that keeps count of the weights, with odd sizes, grouped narrow heads and small pages
        dict(name='weights-decode-5x1037', op='weights', batch=5, new=1, kv=1037, heads=12, kv_heads=3, dim=64, page=16),
        # prefill of a 2-D batch that starts the count
        dict(name='weights-prefill-8x456', op='weights', batch=8, new=456, kv=456, **lm),
        # one conversation cut by a few tokens: latency
        dict(name='evict-1x600-to-512', op='evict', batch=1, kv=600, budget=512, recent=64, **lm),
        # eight volumes cut to a quarter after prefill
        dict(name='evict-8x4609-to-1152', op='evict', batch=8, kv=4609, budget=1152, recent=128, **lm),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """one more case of the same ranges; no dearer than the dearest listed case of its operator"""
    while True:
        op = rng.choice(['append', 'attn', 'attn', 'weights', 'evict'])
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        group = rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv_heads <= 32])
        case = dict(op=op, batch=_log(rng, 1, 32), kv=_log(rng, 1, 16384), heads=kv_heads * group, kv_heads=kv_heads,
                    dim=rng.choice([32, 64, 128, 128]), page=rng.choice([16, 32, 64, 128, 256]))
        if op == 'evict':
            case['budget'] = _log(rng, 1, case['kv'])
            case['recent'] = rng.choice([0, case['budget'] // 8, case['budget'] // 2])
        else:
            case['new'] = rng.choice([1, _log(rng, 1, min(4609, case['kv'])), min(4609, case['kv'])])
            case['packed'] = op != 'append' and rng.random() < 0.5
        cap = [work(c) for c in listed() if c['op'] == op]
        w = work(case)
        if w['bytes'] <= max(c['bytes'] for c in cap) and w['flops'] <= max(c['flops'] for c in cap):
            return case


def _lens(case):
    """(cached tokens, new tokens) of every sample: ragged, the first one the longest; the new ones are counted in the cached ones"""
    b, out = case['batch'], []
    for i in range(b):
        n = max(1, case['kv'] - (case['kv'] // 2) * i // b - (i % 3 if i else 0))
        out.append((n, min(n, max(1, case.get('new', 0) - (case.get('new', 0) // 2) * i // b)) if case['op'] != 'evict' else 0))
    return out


def work(case):
    H, Hk, D = case['heads'], case['kv_heads'], case['dim']
    lens = _lens(case)
    new = sum(n for _, n in lens)
    kept = [min(n, case.get('budget', n)) for n, _ in lens]
    if case['op'] == 'append':
        move = 2 * new * D * (H + 2 * Hk)
        return {'bytes': 2 * move + new * (8 * D + 12), 'flops': 3 * new * D * (H + Hk)}
    if case['op'] == 'evict':
        return {'bytes': Hk * (4 * sum(n for n, _ in lens) + sum(k * (2 * (4 * D + 4) + 4) for k in kept)), 'flops': Hk * sum(n for n, _ in lens)}
    pairs = H * sum(n * (n + 1) // 2 + n * (L - n) for L, n in lens)
    w = {'bytes': 4 * D * H * new + 4 * H * new + 4 * D * Hk * sum(L for L, _ in lens), 'flops': 4 * D * pairs}
    if case['op'] == 'weights':
        w['bytes'] += 8 * Hk * sum(L for L, _ in lens)
        w['flops'] += pairs
    return w


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    B, H, Hk, D, S = case['batch'], case['heads'], case['kv_heads'], case['dim'], case['page']
    lens = _lens(case)
    kv_host, new_host = [a for a, _ in lens], [n for _, n in lens]
    per = -(-max(kv_host) // S)
    kept = [min(n, case.get('budget', 0)) for n in kv_host]
    per_new = -(-max(kept) // S)
    n_old = sum(-(-n // S) for n in kv_host)
    n_new = sum(-(-n // S) for n in kept)
    pages = n_old + n_new + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
    table, new_table, at = torch.full((B, per), -1, dtype=torch.int32), torch.full((B, max(per_new, 1)), -1, dtype=torch.int32), 0
    for t, ns in ((table, kv_host), (new_table, kept)):
        for b, n in enumerate(ns):
            c = -(-n // S)
            t[b, :c] = order[at:at + c]
            at += c
    i32 = dict(dtype=torch.int32, device=DEV)
    st = dict(case=case, kv_host=kv_host, new_host=new_host, table=table.to(DEV), lens=torch.tensor(kv_host, **i32), scale=D ** -0.5)
    shape = (pages, Hk, S, D)
    if case['op'] == 'append':
        T = sum(new_host)
        st['k'], st['v'] = torch.zeros(shape, dtype=torch.bfloat16, device=DEV), torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        st['qkv'] = torch.randn(T, (H + 2 * Hk) * D, generator=g, device=DEV).to(torch.bfloat16)
        seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(new_host)])
        idx = torch.cat([torch.arange(L - n, L, dtype=torch.int32) for L, n in lens])
        st['row_seq'], st['row_idx'] = seq.to(DEV), idx.to(DEV)
        # positions run behind the index (image tokens share one): a gap that grows along the sequence
        st['row_pos'] = (idx - idx // 3).to(DEV)
        inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, device=DEV) / D))
        ang = torch.arange(max(kv_host), device=DEV)[:, None] * torch.cat([inv, inv])[None]
        st['cos'], st['sin'] = ang.cos().contiguous(), ang.sin().contiguous()
        return st
    st['k'] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    st['v'] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    if case['op'] == 'evict':
        w = torch.randn(B, Hk, max(kv_host), generator=g, device=DEV).mul(2).exp()
        w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.2, torch.zeros_like(w), w)     # many tokens nobody looked at: ties
        st['w'] = torch.where(torch.arange(max(kv_host), device=DEV) < st['lens'][:, None, None], w, torch.zeros_like(w)).contiguous()
        st['new_table'] = new_table.to(DEV)
        return st
    T = sum(new_host)
    st['q'] = torch.randn(T, H * D, generator=g, device=DEV).mul(2).to(torch.bfloat16)
    cu = [0]
    for n in new_host:
        cu.append(cu[-1] + n)
    st['cu'] = torch.tensor(cu, **i32)
    st['row_of_pos'] = torch.randperm(T, generator=g, device=DEV).to(torch.int32) if case.get('packed') else None
    if case['op'] == 'weights':
        w = torch.rand(B, Hk, max(kv_host), generator=g, device=DEV)
        st['w'] = torch.where(torch.arange(max(kv_host), device=DEV) < st['lens'][:, None, None], w, torch.zeros_like(w)).contiguous()
        st['w_out'] = torch.zeros_like(st['w'])
    return st


# ---------------------------------------------------------------- one pass
def run(st):
    op = st['case']['op']
    if own:
        from mmmm_amd import kernels as K
        c = st['case']
        if op == 'append':
            q = K.kv_append_paged(st['qkv'], st['row_seq'], st['row_idx'], st['table'], st['k'], st['v'], st['row_pos'], st['cos'], st['sin'], c['heads'])
            return q, st['k'], st['v']
        if op == 'evict':
            w, lens, kept = K.kv_evict_paged(st['k'], st['v'], st['w'], st['table'], st['lens'], st['new_table'], c['budget'], c['recent'])
            return st['k'], st['v'], w, lens, kept
        extra = dict(weights=st['w'], weights_out=st['w_out']) if op == 'weights' else {}
        out, lse = K.attn_paged(st['q'], st['k'], st['v'], st['table'], st['cu'], st['lens'], st['scale'], max(st['new_host']), max(st['kv_host']),
                                row_of_pos=st['row_of_pos'], **extra)
        return (out, lse, st['w_out']) if op == 'weights' else (out, lse)
    if op == 'append':
        return _plain_append(st)
    if op == 'evict':
        return _plain_evict(st)
    return _plain_attention(st)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _plain_append(st):
    c = st['case']
    H, Hk, D, S = c['heads'], c['kv_heads'], c['dim'], c['page']
    x = st['qkv'].float().view(-1, H + 2 * Hk, D)
    pos = st['row_pos'].long()
    cos, sin = st['cos'][pos][:, None], st['sin'][pos][:, None]
    idx = st['row_idx'].long()
    page, off = st['table'][st['row_seq'].long(), idx // S].long(), idx % S
    st['k'][page, :, off] = _rotate(x[:, H:H + Hk], cos, sin).to(torch.bfloat16)
    st['v'][page, :, off] = x[:, H + Hk:].to(torch.bfloat16)
    return _rotate(x[:, :H], cos, sin).reshape(-1, H * D).to(torch.bfloat16), st['k'], st['v']


def _plain_attention(st):
    c = st['case']
    H, Hk, D, S = c['heads'], c['kv_heads'], c['dim'], c['page']
    G = H // Hk
    out, lse = torch.zeros(st['q'].shape, dtype=torch.bfloat16, device=DEV), torch.empty(H, st['q'].shape[0], device=DEV)
    p0 = 0
    for b, (L, n) in enumerate(zip(st['kv_host'], st['new_host'])):
        rows = st['row_of_pos'][p0:p0 + n].long() if st['row_of_pos'] is not None else slice(p0, p0 + n)
        pg = st['table'][b, :-(-L // S)].long()
        k = st['k'][pg].float().permute(1, 0, 2, 3).reshape(Hk, -1, D)[:, :L]
        v = st['v'][pg].float().permute(1, 0, 2, 3).reshape(Hk, -1, D)[:, :L]
        q = st['q'][rows].float().view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(st['scale']).view(Hk, G, n, L)
        hidden = torch.arange(L, device=DEV)[None] > torch.arange(L - n, L, device=DEV)[:, None]
        s.masked_fill_(hidden, float('-inf'))
        m = s.amax(-1, keepdim=True)
        s.sub_(m).exp_()
        z = s.sum(-1, keepdim=True)
        s.div_(z)
        o = torch.bmm(s.view(Hk, G * n, L), v.contiguous()).view(Hk, G, n, D)
        out[rows] = o.permute(2, 0, 1, 3).reshape(n, H * D).to(torch.bfloat16)
        lse[:, p0:p0 + n] = (m + z.log()).view(H, n)
        if c['op'] == 'weights':
            st['w_out'][b, :, :L] = st['w'][b, :, :L] + s.sum((1, 2))
        p0 += n
    return (out, lse, st['w_out']) if c['op'] == 'weights' else (out, lse)


def _plain_evict(st):
    c = st['case']
    S, budget, recent, Hk = c['page'], c['budget'], c['recent'], c['kv_heads']
    w = st['w']
    B = w.shape[0]
    w_new, kept = torch.zeros_like(w), torch.full((B, Hk, budget), -1, dtype=torch.int32, device=DEV)
    heads = torch.arange(Hk, device=DEV)[:, None]
    for b, L in enumerate(st['kv_host']):
        n = min(L, budget)
        score = w[b, :, :L].clone()
        score[:, L - min(recent, n):] = float('inf')
        idx = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :n].sort(dim=1).values
        kept[b, :, :n] = idx.to(torch.int32)
        w_new[b, :, :n] = w[b].gather(1, idx)
        src = st['table'][b].long()[idx // S]
        at = torch.arange(n, device=DEV)
        dst = st['new_table'][b].long()[at // S][None]
        st['k'][dst, heads, (at % S)[None]] = st['k'][src, heads, idx % S]
        st['v'][dst, heads, (at % S)[None]] = st['v'][src, heads, idx % S]
    return st['k'], st['v'], w_new, st['lens'].clamp(max=budget), kept


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    H, Hk, D, S = case['heads'], case['kv_heads'], case['dim'], case['page']
    f64 = torch.float64
    if case['op'] == 'append':
        T = st['qkv'].shape[0]
        k, v, q = st['k'].to(f64), st['v'].to(f64), torch.empty(T, H * D, dtype=f64, device=DEV)
        x = st['qkv'].view(T, H + 2 * Hk, 2, D // 2)
        pos = st['row_pos'].long()
        c, s = (st[n].view(-1, 2, D // 2)[pos].to(f64) for n in ('cos', 'sin'))
        page = st['table'][st['row_seq'].long(), torch.div(st['row_idx'], S, rounding_mode='floor').long()].long()
        off = (st['row_idx'] % S).long()
        for h in range(H + Hk):
            lo, hi = x[:, h, 0].to(f64), x[:, h, 1].to(f64)
            y = torch.cat([lo * c[:, 0] - hi * s[:, 0], hi * c[:, 1] + lo * s[:, 1]], 1)
            if h < H:
                q[:, h * D:(h + 1) * D] = y
            else:
                k[page, h - H, off] = y
                v[page, h - H, off] = st['qkv'][:, (h + Hk) * D:(h + Hk + 1) * D].to(f64)
        return q, k, v
    if case['op'] == 'evict':
        budget = case['budget']
        k, v, w = st['k'].to(f64), st['v'].to(f64), torch.zeros(st['w'].shape, dtype=f64, device=DEV)
        kept = torch.full((case['batch'], Hk, budget), -1, dtype=torch.int32, device=DEV)
        for b, L in enumerate(st['kv_host']):
            n = min(L, budget)
            fixed = min(case['recent'], n)
            for h in range(Hk):
                old = st['w'][b, h, :L - fixed].cpu().tolist()
                best = sorted(range(len(old)), key=lambda j: (-old[j], j))[:n - fixed]
                keep = torch.tensor(sorted(best) + list(range(L - fixed, L)), device=DEV)
                kept[b, h, :n] = keep.to(torch.int32)
                w[b, h, :n] = st['w'][b, h][keep].to(f64)
                at = torch.arange(n, device=DEV)
                src, dst = st['table'][b].long()[keep // S], st['new_table'][b].long()[at // S]
                k[dst, h, at % S] = st['k'][src, h, keep % S].to(f64)
                v[dst, h, at % S] = st['v'][src, h, keep % S].to(f64)
        return k, v, w, torch.tensor([min(L, budget) for L in st['kv_host']], dtype=torch.int32, device=DEV), kept
    T = st['q'].shape[0]
    out, lse = torch.zeros(T, H, D, dtype=f64, device=DEV), torch.zeros(H, T, dtype=f64, device=DEV)
    w = st['w'].to(f64) if case['op'] == 'weights' else None
    rows = st['row_of_pos'].long() if st['row_of_pos'] is not None else torch.arange(T, device=DEV)
    p0 = 0
    for b, (L, n) in enumerate(zip(st['kv_host'], st['new_host'])):
        j = torch.arange(L, device=DEV)
        page, off = st['table'][b].long()[j // S], j % S
        seen = j[None] <= (L - n + torch.arange(n, device=DEV))[:, None]
        for h in range(H):
            kh, vh = st['k'][page, h * Hk // H, off].to(f64), st['v'][page, h * Hk // H, off].to(f64)
            s = (st['q'][rows[p0:p0 + n], h * D:(h + 1) * D].to(f64) * st['scale']) @ kh.T.contiguous()
            z = torch.logsumexp(torch.where(seen, s, float('-inf')), 1)
            p = torch.where(seen, torch.exp(s - z[:, None]), 0.0)
            out[rows[p0:p0 + n], h] = p @ vh
            lse[h, p0:p0 + n] = z
            if w is not None:
                w[b, h * Hk // H, :L] += p.sum(0)
        p0 += n
    return (out.view(T, H * D), lse, w) if w is not None else (out.view(T, H * D), lse)
