"""Paged-cache operators on the MI355X against their 64-bit statements (tests/_paged.py), elementwise, with tolerances that count the
roundings. Rows of the pools that hold no token are NaN throughout: nothing may read them as data."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests import _paged as R

pytestmark = pytest.mark.gpu
NAN = float('nan')


@pytest.fixture(scope='module')
def K():
    from mmmm_amd import kernels
    return kernels


def close(got, want, tol, what=''):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isfinite(), want.isfinite()), what
    fin = want.isfinite()
    assert torch.equal(got[~fin], want[~fin]), what
    err = (got[fin] - want[fin]).abs() - tol[fin]
    assert err.numel() == 0 or float(err.max()) <= 0, (what, float(err.max()), float((got[fin] - want[fin]).abs().max()))


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def run_attention(K, dev, new, lens, H, hk, hd, page, packed=False, weights=False, seed=0, absent=(), scale=None, cols=None, qs=1.5):
    g = torch.Generator().manual_seed(seed)
    k, v, table = R.make_cache(lens, hk, hd, page, g, cols=cols)
    for b, c, val in absent:
        table[b, c] = val
    T = sum(new)
    rows = T + 5                                                          # rows of no position behind the last one
    q = (torch.randn(rows, H * hd, generator=g) * qs).bfloat16()
    rop = torch.randperm(rows, generator=g)[:rows].to(torch.int32) if packed else None
    scale = hd ** -0.5 if scale is None else scale
    w = torch.rand(len(lens), hk, max(1, max(lens)) + 3, generator=g) if weights else None
    want = R.attention(q, k, v, table, new, lens, scale, rop, w)
    big = torch.full((rows, H * hd + 24), 7.0, dtype=torch.bfloat16, device=dev)      # strided q and out
    big[:, 8:8 + H * hd] = q.to(dev)
    out = torch.full((rows, H * hd + 8), 3.0, dtype=torch.bfloat16, device=dev)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    kw = {}
    if weights:
        wd = w.to(dev)
        wo = torch.full_like(wd, -1.0)
        kw = dict(weights=wd, weights_out=wo)
    args = (big[:, 8:8 + H * hd], k.to(dev), v.to(dev), table.to(dev), i32(cu, dev), i32(lens, dev), scale, max(new), max(lens))
    o, lse = K.attn_paged(*args, row_of_pos=rop.to(dev) if packed else None, out=out[:, :H * hd], **kw)
    pos = torch.arange(T)
    r = rop.long()[pos] if packed else pos
    close(o.cpu()[r], want[0][r], want[1][r], 'out')
    close(lse.cpu()[:, :T], want[2][:, :T], want[3][:, :T], 'lse')
    rest = torch.ones(rows, dtype=torch.bool)
    rest[r] = False
    assert (o.cpu()[rest] == 3.0).all() and (out[:, H * hd:] == 3.0).all()            # left as they were
    if weights:
        for b, L in enumerate(lens):
            close(wo[b, :, :L], want[4][b, :, :L], want[5][b, :, :L], 'weights')
            assert (wo[b, :, L:] == -1.0).all()
        assert torch.equal(wd.cpu(), w)
    o2, lse2 = K.attn_paged(*args, row_of_pos=rop.to(dev) if packed else None, **kw)
    assert torch.equal(o2.cpu()[r], o.cpu()[r]) and torch.equal(lse2[:, :T], lse[:, :T])      # same bits again
    return o


# (new tokens, cached tokens), query heads, kv heads, width, page
ATTN = [
    ([1], [1], 1, 1, 128, 16),
    ([1, 1, 1], [1, 64, 65], 4, 4, 128, 64),
    ([1, 1, 1, 1], [485, 31, 2, 257], 3, 3, 128, 32),
    ([1, 1], [1000, 777], 8, 1, 64, 16),
    ([1, 1], [300, 1], 12, 3, 32, 256),
    ([2, 1, 5], [130, 7, 5], 6, 2, 128, 128),
    ([7, 0, 3], [40, 0, 3], 2, 2, 64, 16),
    ([16, 17], [16, 400], 4, 2, 128, 64),
    ([33, 64], [97, 64], 2, 1, 32, 32),
    ([37, 30, 1], [2086, 200, 90], 2, 2, 128, 64),
    ([100, 65], [100, 321], 4, 1, 128, 16),
    ([129, 257], [129, 300], 3, 3, 128, 64),
    ([300], [300], 8, 2, 64, 128),
    ([513], [1200], 2, 1, 128, 64),
    ([200, 310], [456, 310], 2, 2, 32, 1024),
]


@pytest.mark.parametrize('case', ATTN, ids=[str(i) for i in range(len(ATTN))])
@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('weights', [False, True])
def test_attention(dev, K, case, packed, weights):
    run_attention(K, dev, *case, packed=packed, weights=weights, seed=len(case[0]))


@pytest.mark.parametrize('new,lens', [([1], [5000]), ([3], [9001]), ([40], [3000]), ([70, 1], [4097, 1])])
def test_attention_long_cache(dev, K, new, lens):
    run_attention(K, dev, new, lens, 4, 2, 128, 64, packed=True, weights=True)


@pytest.mark.parametrize('new,lens', [([5, 2], [3, 0]), ([40], [7]), ([300, 1], [270, 0])])
@pytest.mark.parametrize('hd', [64, 128])
def test_rows_that_see_nothing(dev, K, new, lens, hd):
    """more new tokens than cached ones: the first of them see no token at all -> zeros, lse -inf"""
    run_attention(K, dev, new, lens, 4, 2, hd, 16, weights=True)


@pytest.mark.parametrize('new', [1, 9, 80, 300])
@pytest.mark.parametrize('page', [16, 64, 256])
def test_absent_pages_are_masked(dev, K, new, page):
    """first, middle and last pages missing (-1, far out of range): never read through, their tokens are not there"""
    absent = [(0, 0, -1), (0, 1, 2 ** 31 - 1), (1, 0, -2 ** 31), (0, 512 // page - 1, 10 ** 6)]
    run_attention(K, dev, [new, min(new, 100)], [512, 300], 2, 1, 128, page, weights=True, absent=absent)
    run_attention(K, dev, [new], [min(512, page)], 2, 2, 64, page, absent=[(0, 0, -7)]) if new <= page else None      # nothing left at all


def test_large_scores(dev, K):
    """scores of hundreds: the running maximum has to move, and nothing may overflow"""
    for new in (1, 20, 200):
        run_attention(K, dev, [new], [700], 2, 1, 128, 64, weights=True, qs=60.0)


def test_other_scale(dev, K):
    for new in (1, 70):
        run_attention(K, dev, [new], [333], 2, 2, 128, 64, scale=0.7)


def test_attention_of_nothing(dev, K):
    g = torch.Generator().manual_seed(0)
    k, v, table = (t.to(dev) for t in R.make_cache([40], 2, 64, 16, g))
    q = torch.zeros(0, 2 * 64, dtype=torch.bfloat16, device=dev)
    o, lse = K.attn_paged(q, k, v, table, i32([0, 0], dev), i32([40], dev), 0.1, 0, 40)
    assert o.shape == (0, 128) and lse.shape == (2, 0)
    w = torch.rand(1, 2, 48, generator=g).to(dev)
    wo = torch.full_like(w, -1.0)
    K.attn_paged(q, k, v, table, i32([0, 0], dev), i32([40], dev), 0.1, 0, 40, weights=w, weights_out=wo)
    assert torch.equal(wo[..., :40], w[..., :40]) and (wo[..., 40:] == -1.0).all()


@pytest.mark.parametrize('hd', [32, 64, 128])
@pytest.mark.parametrize('H,hk,page', [(1, 1, 16), (32, 32, 64), (6, 2, 256), (5, 5, 32)])
def test_append(dev, K, hd, H, hk, page):
    g = torch.Generator().manual_seed(hd + H)
    lens = [page * 2 + 3, 1, 70]
    k, v, table = R.make_cache(lens, hk, hd, page, g, poison=False)
    table[2, 0] = -1                                                        # a page that is not there
    rows = []
    for b, L in enumerate(lens):
        rows += [(b, j) for j in range(max(0, L - 40), L)]
    rows += [(-1, 0), (3, 0), (0, -1), (0, table.shape[1] * page), (2 ** 31 - 1, 5)]      # not stored
    rows = [rows[i] for i in torch.randperm(len(rows), generator=g).tolist()]
    T = len(rows)
    seq, idx = (torch.tensor(c, dtype=torch.int32) for c in zip(*rows))
    pos = torch.randint(-2, 60, (T,), generator=g).to(torch.int32)           # clamped to the table
    n_pos = 50
    ang = torch.rand(n_pos, hd, generator=g) * 6
    cos, sin = ang.cos(), ang.sin()
    qkv = torch.randn(T + 2, (H + 2 * hk) * hd + 8, generator=g).bfloat16()
    for nrows in (None, T - 7):
        n = T if nrows is None else nrows
        want = R.append(qkv[:n, :(H + 2 * hk) * hd].contiguous(), seq[:n], idx[:n], table, k, v, pos[:n], cos, sin, H)
        kd, vd, x = k.to(dev), v.to(dev), qkv.to(dev)
        q = torch.full((T + 1, H * hd), 5.0, dtype=torch.bfloat16, device=dev)
        K.kv_append_paged(x[:T, :(H + 2 * hk) * hd], seq.to(dev), idx.to(dev), table.to(dev), kd, vd, pos.to(dev), cos.to(dev), sin.to(dev), H,
                          nrows=None if nrows is None else i32([nrows], dev), q_out=q[:T])
        close(q[:n], want[0], want[1], 'q')
        close(kd, want[2], want[3], 'k')
        assert torch.equal(vd.cpu().double(), want[4])
        assert (q[n:] == 5.0).all() and torch.equal(x.cpu(), qkv)


@pytest.mark.parametrize('lens,budget,recent', [([600], 512, 64), ([1, 0, 40], 8, 8), ([5000, 33, 512], 100, 0), ([64, 65, 66], 64, 1), ([300, 20], 1, 0),
                                                ([2100], 2099, 700)])
@pytest.mark.parametrize('hd,hk,page', [(128, 3, 64), (32, 1, 16)])
@pytest.mark.parametrize('kind', ['random', 'ties', 'odd'])
def test_evict(dev, K, lens, budget, recent, hd, hk, page, kind):
    g = torch.Generator().manual_seed(sum(lens) + budget)
    both = list(lens) + [min(n, budget) for n in lens]                       # old pages and new ones from one pool
    k, v, tab = R.make_cache(both, hk, hd, page, g)
    table, new_table = tab[:len(lens)], tab[len(lens):].clone()
    cols = max(lens) + 2
    w = torch.rand(len(lens), hk, cols, generator=g)
    if kind == 'ties':
        w = (w * 3).floor()
    if kind == 'odd':
        w = torch.where(w < 0.2, NAN, torch.where(w < 0.4, float('-inf'), torch.where(w < 0.5, -0.0, torch.where(w < 0.6, 0.0, torch.where(w > 0.97, float('inf'), -w)))))
        if max(lens) > page:
            table[0, 0] = -1
            table[len(lens) - 1, 0] = 2 ** 30
    kept, new = R.evict(w, table, k.shape[0], page, lens, budget, recent)
    kd, vd = k.to(dev), v.to(dev)
    got_w, got_l, got_k = K.kv_evict_paged(kd, vd, w.to(dev), table.to(dev), i32(lens, dev), new_table.to(dev), budget, recent)
    assert got_l.cpu().tolist() == new
    ke, ve = k.clone(), v.clone()
    for b in range(len(lens)):
        for h in range(hk):
            idx = torch.tensor(kept[b][h], dtype=torch.long)
            n = len(idx)
            assert got_k[b, h].cpu().tolist() == idx.tolist() + [-1] * (budget - n)
            a, c = got_w[b, h].cpu(), w[b, h][idx]
            assert torch.equal(a[:n].view(torch.int32), c.view(torch.int32)) and (a[n:] == 0).all()
            at = torch.arange(n)
            src, dst = table[b].long()[idx // page], new_table[b].long()[at // page]
            ke[dst, h, at % page], ve[dst, h, at % page] = k[src, h, idx % page], v[src, h, idx % page]
    assert torch.equal(kd.cpu().view(torch.int16), ke.view(torch.int16)) and torch.equal(vd.cpu().view(torch.int16), ve.view(torch.int16))


def test_append_attend_evict_together(dev, K):
    """a conversation as the cache lives it: prompt, follow-up, single tokens, eviction, more tokens — against the same in 64 bits"""
    g = torch.Generator().manual_seed(11)
    H, hk, hd, page, B = 4, 2, 64, 16, 2
    pages = 64
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table, free = torch.full((B, 12), -1, dtype=torch.int32), perm.tolist()
    for b in range(B):
        table[b, :12] = torch.tensor([free.pop() for _ in range(12)], dtype=torch.int32)
    k = torch.full((pages, hk, page, hd), NAN).bfloat16()
    v = k.clone()
    kd, vd = k.to(dev), v.to(dev)
    ang = torch.arange(256)[:, None] * torch.cat([1.0 / 10000 ** (torch.arange(0, hd, 2) / hd)] * 2)[None]
    cos, sin = ang.cos(), ang.sin()
    lens, w, wd = [0, 0], torch.zeros(B, hk, 192), torch.zeros(B, hk, 192, device=dev)
    seen = [0, 0]
    for step, new in enumerate([[100, 71], [9, 20], [1, 1], [1, 1], 'evict', [1, 1], [30, 2]]):
        if new == 'evict':
            nt = torch.full((B, 12), -1, dtype=torch.int32)
            for b in range(B):
                nt[b] = torch.tensor([free.pop() for _ in range(12)], dtype=torch.int32)
            kept, new_lens = R.evict(wd.cpu(), table, pages, page, lens, 48, 8)           # the choice is exact given the weights
            wd2, ld, got = K.kv_evict_paged(kd, vd, wd, table.to(dev), i32(lens, dev), nt.to(dev), 48, 8)
            assert ld.cpu().tolist() == new_lens
            k2, v2, w2 = k.clone(), v.clone(), torch.zeros_like(w)
            for b in range(B):
                for h in range(hk):
                    idx = torch.tensor(kept[b][h])
                    assert got[b, h].cpu().tolist() == kept[b][h]
                    at = torch.arange(len(idx))
                    k2[nt[b].long()[at // page], h, at % page] = k[table[b].long()[idx // page], h, idx % page]
                    v2[nt[b].long()[at // page], h, at % page] = v[table[b].long()[idx // page], h, idx % page]
                    w2[b, h, :len(idx)] = w[b, h][idx]
            k, v, w, wd, table, lens = k2, v2, w2, wd2, nt, new_lens
            continue
        T = sum(new)
        qkv = torch.randn(T, (H + 2 * hk) * hd, generator=g).bfloat16()
        rows = [(b, lens[b] + i, seen[b] + i) for b in range(B) for i in range(new[b])]
        seq, idx, pos = (torch.tensor(c, dtype=torch.int32) for c in zip(*rows))
        lens = [a + n for a, n in zip(lens, new)]
        seen = [a + n for a, n in zip(seen, new)]
        q = K.kv_append_paged(qkv.to(dev), seq.to(dev), idx.to(dev), table.to(dev), kd, vd, pos.to(dev), cos.to(dev), sin.to(dev), H)
        qw, qt, kw, kt, vw = R.append(qkv, seq, idx, table, k, v, pos, cos, sin, H)
        close(q, qw, qt)
        for b in range(B):
            for h in range(hk):
                close(R.tokens(kd.cpu(), table, b, lens[b], h)[0], R.tokens(kw, table, b, lens[b], h)[0], R.tokens(kt, table, b, lens[b], h)[0])
        k, v = kd.cpu(), vd.cpu()                                                        # what was stored is the next stage's input
        cu = [0, new[0], T]
        want = R.attention(q.cpu(), k, v, table, new, lens, hd ** -0.5, None, wd.cpu())
        o, lse = K.attn_paged(q, kd, vd, table.to(dev), i32(cu, dev), i32(lens, dev), hd ** -0.5, max(new), max(lens), weights=wd)
        close(o, want[0], want[1], f'step {step}')
        close(lse, want[2], want[3])
        close(wd, want[4], want[5])
        w = wd.cpu()


@pytest.mark.parametrize('new,L', [(4, 40), (13, 13), (37, 100), (200, 330), (300, 300)])
@pytest.mark.parametrize('hd', [32, 128])
def test_what_a_query_does_not_see_does_not_reach_it(dev, K, new, L, hd):
    """inf and NaN in keys and values of LATER tokens of the chunk: earlier queries do not notice, later ones get what arithmetic gives"""
    g = torch.Generator().manual_seed(new)
    H, hk, page = 4, 2, 16
    k, v, table = R.make_cache([L], hk, hd, page, g)
    q = torch.randn(new, H * hd, generator=g).bfloat16()
    bad = [L - 1, L - new // 3 - 1, L - new // 2 - 1]
    for n, (j, x) in enumerate(zip(bad, (NAN, float('inf'), -float('inf')))):
        v[int(table[0, j // page]), n % hk, j % page, 3 * n:3 * n + 5] = x
    kb = L - 1
    k[int(table[0, kb // page]), 1, kb % page, 7] = NAN                      # the newest key too: only the last query sees it
    w = torch.zeros(1, hk, L)
    clean_k, clean_v = k.nan_to_num(0.0, 0.0, 0.0), v.nan_to_num(0.0, 0.0, 0.0)
    scale = hd ** -0.5
    want = R.attention(q, clean_k, clean_v, table, [new], [L], scale, None, w)
    dt = table.to(dev)
    out, lse = K.attn_paged(q.to(dev), k.to(dev), v.to(dev), dt, i32([0, new], dev), i32([L], dev), scale, new, L)
    got = out.cpu().double().view(new, H, hd)
    ref, tol = want[0].view(new, H, hd), want[1].view(new, H, hd)
    touched = torch.zeros(new, H, hd, dtype=torch.bool)
    kind = torch.zeros(new, H, hd)
    for n, j in enumerate(bad):
        i0 = j - (L - new)                                                   # the first query that sees token j
        heads = slice(2 * (n % hk), 2 * (n % hk) + 2)
        touched[i0:, heads, 3 * n:3 * n + 5] = True
        kind[i0:, heads, 3 * n:3 * n + 5] += n
    touched[new - 1, 2:] = True                                              # NaN score: the whole row
    assert ((got - ref).abs() <= tol)[~touched].all()
    assert (~got.isfinite())[touched].all()
    for n, sign in ((1, 1), (2, -1)):
        i0, heads = bad[n] - (L - new), slice(2 * (n % hk), 2 * (n % hk) + 2)
        part = got[i0:new - 1, heads, 3 * n + 3:3 * n + 5] if n == 1 else got[i0:new - 1, heads, 8:11]
        assert (part == sign * float('inf')).all(), n


def _case(K, dev, new, L, seed, H=4, hk=2, hd=128, page=64, weights=False):
    g = torch.Generator().manual_seed(seed)
    k, v, table = R.make_cache([L, max(1, L // 2)], hk, hd, page, g)
    n2 = min(new, max(1, L // 2))
    q = torch.randn(new + n2, H * hd, generator=g).bfloat16().to(dev)
    args = [q, k.to(dev), v.to(dev), table.to(dev), i32([0, new, new + n2], dev), i32([L, max(1, L // 2)], dev), hd ** -0.5, new, L]
    kw = dict(weights=torch.rand(2, hk, L, generator=g).to(dev)) if weights else {}
    if weights:
        kw['weights_out'] = torch.zeros_like(kw['weights'])
    return args, kw


def test_two_captured_graphs_and_eager_calls_between(dev, K):
    """each graph has its own workspace: replays of one do not disturb the other, whatever runs between"""
    cases = [_case(K, dev, 1, 3000, 1, weights=True), _case(K, dev, 50, 2500, 2, weights=True)]
    want = []
    for a, kw in cases:
        o, lse = K.attn_paged(*a, **kw)
        want.append((o.clone(), lse.clone(), kw['weights_out'].clone()))
    torch.cuda.synchronize()
    graphs = []
    for a, kw in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o, lse = K.attn_paged(*a, **kw)
        graphs.append((gr, o, lse, kw['weights_out']))
    for rep in range(4):
        for (gr, o, lse, wo), w in zip(graphs if rep % 2 else graphs[::-1], want if rep % 2 else want[::-1]):
            wo.zero_()
            gr.replay()
            K.attn_paged(*cases[rep % 2][0])
            torch.randn(1 << 16, device=dev).sum()
            torch.cuda.synchronize()
            assert torch.equal(o, w[0]) and torch.equal(lse, w[1]) and torch.equal(wo, w[2])


def test_on_another_stream(dev, K):
    args, kw = _case(K, dev, 40, 2000, 3, weights=True)
    o, lse = K.attn_paged(*args, **kw)
    w = kw['weights_out'].clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        kw['weights_out'].zero_()
        o2, lse2 = K.attn_paged(*args, **kw)
        x = o2 + 0
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(x, o) and torch.equal(lse2, lse) and torch.equal(kw['weights_out'], w)


def test_pools_beyond_32_bit_offsets(dev, K):
    """pages behind 2^31 elements (4 GiB) of a pool: stored, attended to in both forms, moved"""
    g = torch.Generator().manual_seed(4)
    H, hk, hd, page = 16, 8, 128, 1024
    pages = 2 * (1 << 31) // (hk * page * hd) // 2 + 12                       # 2060 pages of 2^20 elements
    assert (pages - 8) * hk * page * hd > 1 << 31
    k = torch.empty(pages, hk, page, hd, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 1, 3, pages - 4]], dtype=torch.int32)
    L = 2 * page + 300
    qkv = torch.randn(L, (H + 2 * hk) * hd, generator=g).bfloat16()
    ang = torch.rand(16, hd, generator=g)
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, 16, (L,), generator=g).to(torch.int32)
    seq, idx = torch.zeros(L, dtype=torch.int32), torch.arange(L, dtype=torch.int32)
    q = K.kv_append_paged(qkv.to(dev), seq.to(dev), idx.to(dev), table.to(dev), k, v, pos.to(dev), cos.to(dev), sin.to(dev), H)
    few = [pages - 1, 3, pages - 4]
    ks, vs, small = k[few].cpu(), v[few].cpu(), torch.tensor([[0, 1, 2]], dtype=torch.int32)
    z = torch.zeros(3, hk, page, hd, dtype=torch.bfloat16)
    qw, qt, kw, kt, vw = R.append(qkv, seq, idx, small, z, z, pos, cos, sin, H)
    close(q, qw, qt)
    for h in range(hk):
        close(R.tokens(ks, small, 0, L, h)[0], R.tokens(kw, small, 0, L, h)[0], R.tokens(kt, small, 0, L, h)[0])
        assert torch.equal(R.tokens(vs, small, 0, L, h)[0], R.tokens(vw, small, 0, L, h)[0])
    for n in (1, 64):
        qn = q[-n:].contiguous()
        want = R.attention(qn.cpu(), ks, vs, small, [n], [L], hd ** -0.5)
        o, lse = K.attn_paged(qn, k, v, table.to(dev), i32([0, n], dev), i32([L], dev), hd ** -0.5, n, L)
        close(o, want[0], want[1])
        close(lse, want[2], want[3])
    w = torch.rand(1, hk, L, generator=g)
    new = torch.tensor([[pages - 7]], dtype=torch.int32)
    kept, lens = R.evict(w, table, pages, page, [L], 900, 10)
    _, _, got = K.kv_evict_paged(k, v, w.to(dev), table.to(dev), i32([L], dev), new.to(dev), 900, 10)
    for h in range(hk):
        assert got[0, h].cpu().tolist() == kept[0][h]
        i = torch.tensor(kept[0][h])
        assert torch.equal(k[pages - 7, h, :900].cpu(), ks[(i // page), h, i % page])
        assert torch.equal(v[pages - 7, h, :900].cpu(), vs[(i // page), h, i % page])


def test_strides_of_the_pools_and_tables(dev, K):
    """K and V of a layer interleaved in one allocation, tables and weights that are views"""
    g = torch.Generator().manual_seed(8)
    lens, hk, hd, page, H = [70, 130], 2, 64, 32, 4
    k, v, table = R.make_cache(lens, hk, hd, page, g)
    both = torch.stack([k, v], 1).to(dev)                                    # [pages, 2, ...]: page stride of two pages
    wide = torch.full((2, 11), -9, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    w = torch.rand(2, hk, 200, generator=g)
    ww = torch.zeros(2, hk + 1, 260)
    ww[:, 1:, 30:230] = w
    q = torch.randn(9, H * hd, generator=g).bfloat16()
    want = R.attention(q, k, v, table, [4, 5], lens, 0.2, None, w)
    wd = ww.to(dev)
    o, lse = K.attn_paged(q.to(dev), both[:, 0], both[:, 1], wide.to(dev)[:, 2:2 + table.shape[1]], i32([0, 4, 9], dev), i32(lens, dev), 0.2, 5, 130,
                          weights=wd[:, 1:, 30:230])
    close(o, want[0], want[1])
    for b in range(2):
        close(wd[b, 1:, 30:30 + lens[b]], want[4][b, :, :lens[b]], want[5][b, :, :lens[b]])
    rest = wd.cpu().clone()
    rest[:, 1:, 30:230] = 0
    assert (rest == 0).all()


def test_bounds_that_are_too_small_stay_inside(dev, K):
    """max_q below a sample's new tokens: the first of them are computed, nothing is written elsewhere"""
    g = torch.Generator().manual_seed(6)
    for new, bound in ((30, 5), (300, 100)):
        k, v, table = R.make_cache([400], 2, 64, 16, g)
        q = torch.randn(new, 4 * 64, generator=g).bfloat16()
        want = R.attention(q, k, v, table, [new], [400], 0.1)
        out = torch.full((new, 256), 3.0, dtype=torch.bfloat16, device=dev)
        K.attn_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), i32([0, new], dev), i32([400], dev), 0.1, bound, 400, out=out)
        close(out[:bound], want[0][:bound], want[1][:bound])
        assert ((out[bound:] == 3.0).all(1) | ((out[bound:].cpu().double() - want[0][bound:]).abs() <= want[1][bound:]).all(1).to(dev)).all()


@pytest.mark.parametrize('new', [3, 37, 130])
def test_weights_of_infinite_keys(dev, K, new):
    """a key that no query wants at all (score -inf): it receives nothing, also where the last tile of queries is not full"""
    g = torch.Generator().manual_seed(new)
    k, v, table = R.make_cache([400], 1, 128, 64, g)
    k[int(table[0, 1]), 0, 5, 0] = float('-inf')                             # token 69
    q = torch.randn(new, 2 * 128, generator=g).bfloat16()
    q[:, 0::128] = 1.0
    w = torch.rand(1, 1, 400, generator=g)
    got = w.to(dev)
    out, _ = K.attn_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), i32([0, new], dev), i32([400], dev), 0.1, new, 400, weights=got)
    assert bool(out.isfinite().all()) and bool(got.isfinite().all())
    assert float(got[0, 0, 69]) == float(w[0, 0, 69])
    assert bool((got.cpu()[0, 0, :69] > w[0, 0, :69]).all())


@pytest.mark.parametrize('new', [3, 37])
def test_absent_pages_receive_nothing_from_strange_queries(dev, K, new):
    """a query of NaN gives NaN to every token that it sees, and nothing to a token whose page is not there"""
    g = torch.Generator().manual_seed(new)
    k, v, table = R.make_cache([400], 1, 64, 16, g)
    table[0, 3] = -1
    q = torch.randn(new, 64, generator=g).bfloat16()
    q[1] = NAN
    w = torch.rand(1, 1, 400, generator=g)
    got = w.to(dev)
    K.attn_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), i32([0, new], dev), i32([400], dev), 0.1, new, 400, weights=got)
    got = got.cpu()[0, 0]
    assert torch.equal(got[48:64], w[0, 0, 48:64])
    seen = torch.arange(400) <= 400 - new + 1
    seen[48:64] = False
    assert bool(got[seen].isnan().all()) and bool(got[400 - new + 2:].isfinite().all())


@pytest.mark.parametrize('new', [4, 37, 300])
@pytest.mark.parametrize('L', [600, 5000])
def test_positions_without_a_row(dev, K, new, L):
    """row_of_pos outside the rows: no such query, lse -inf, and it counts nowhere"""
    g = torch.Generator().manual_seed(new)
    k, v, table = R.make_cache([L], 2, 128, 64, g)
    q = torch.randn(new, 4 * 128, generator=g).bfloat16()
    rop = torch.randperm(new, generator=g).to(torch.int32)
    gone = [1, new - 2]
    w = torch.zeros(1, 2, L)
    want = R.attention(q, k, v, table, [new], [L], 0.1, rop, w)
    for n in gone:                                                           # their share of the received weights, taken back
        kk = [R.tokens(k, table, 0, L, h)[0] for h in range(2)]
        for h in range(4):
            x = q[int(rop[n]), h * 128:(h + 1) * 128].double() @ kk[h // 2].T * 0.1
            x[L - new + n + 1:] = float('-inf')
            want[4][0, h // 2] -= torch.softmax(x, 0)
        want[2][:, n] = float('-inf')
    lost = [int(rop[n]) for n in gone]
    rop[gone[0]], rop[gone[1]] = -1, new
    out = torch.full((new, 512), 3.0, dtype=torch.bfloat16, device=dev)
    got = w.to(dev)
    o, lse = K.attn_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), i32([0, new], dev), i32([L], dev), 0.1, new, L, row_of_pos=rop.to(dev),
                          weights=got, out=out)
    keep = torch.ones(new, dtype=torch.bool)
    keep[lost] = False
    assert bool((o.cpu()[~keep] == 3.0).all())
    close(o.cpu()[keep], want[0][keep], want[1][keep])
    close(lse, want[2], want[3])
    close(got, want[4], want[5])


def test_an_empty_batch(dev, K):
    """no sample at all: every entry point does nothing and says so"""
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=dev)
    v, t, none = k.clone(), torch.zeros(0, 3, dtype=torch.int32, device=dev), i32([], dev)
    cs = torch.zeros(8, 64, device=dev)
    w = torch.zeros(0, 2, 48, device=dev)
    q = K.kv_append_paged(torch.zeros(0, 8 * 64, dtype=torch.bfloat16, device=dev), none, none, t, k, v, none, cs, cs, 4)
    o, lse = K.attn_paged(q, k, v, t, i32([0], dev), none, 0.1, 0, 0, weights=w)
    nw, nl, kept = K.kv_evict_paged(k, v, w, t, none, t.clone(), 8, 2)
    assert o.shape == (0, 256) and lse.shape == (4, 0) and nw.shape == w.shape and nl.shape == (0,) and kept.shape == (0, 2, 8)


@pytest.mark.parametrize('new', [[0, 2, 0], [0, 0, 40], [0, 0, 0]])
@pytest.mark.parametrize('lens', [[30, 60, 7], [700, 2000, 90]])
def test_samples_without_new_tokens_keep_their_weights(dev, K, new, lens):
    lens = [max(n, L) for n, L in zip(new, lens)]
    run_attention(K, dev, new, lens, 4, 2, 64, 16, weights=True)


@pytest.mark.parametrize('L,B', [(40, 8), (511, 8), (1200, 40)])
def test_weights_of_single_tokens_of_many_heads(dev, K, L, B):
    """one workgroup per cache: the received weights come from the same launch"""
    run_attention(K, dev, [1 + b % 2 for b in range(B)], [max(2, L - 3 * b) for b in range(B)], 32, 16, 32, 64, weights=True, packed=True)


def test_weights_of_chunks_of_many_heads(dev, K):
    """more blocks of tokens than CUs: one set of waves each"""
    run_attention(K, dev, [150, 200, 129, 1, 70, 200], [333, 200, 300, 280, 270, 257], 16, 16, 64, 32, weights=True, packed=True)
    run_attention(K, dev, [300, 40], [300, 130], 64, 64, 32, 64, weights=True)


def test_no_pages_change_hands_inside_a_capture(dev, K):
    from mmmm_amd.models.cogvlm.kv_cache import PagedKVCache
    cache = PagedKVCache(1, 2, 256, 2, 64, dev, page_size=16, n_pages=64, track_weights=True)
    cache.reserve(40)
    cache.len_bound = 40
    free, table = cache.free_pages, cache.block_table.clone()
    x = torch.zeros(4, device=dev)
    for call in (lambda: cache.reserve(100), lambda: cache.evict(8, 2)):
        with pytest.raises(RuntimeError, match='captured'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                x.add_(1)
                call()
        assert cache.free_pages == free and torch.equal(cache.block_table, table)


FIRST_CALL = """
import torch
from mmmm_amd import kernels as K
dev = torch.device('cuda', 0)
g = torch.Generator().manual_seed(0)
k, v = (torch.randn(16, 2, 64, 128, generator=g).bfloat16().to(dev) for _ in range(2))
t = torch.arange(14, dtype=torch.int32, device=dev).view(2, 7)
nt = t.flip(1).contiguous() + 2
q = torch.randn(400, 4 * 128, generator=g).bfloat16().to(dev)
cu, lens = torch.tensor([0, 300, 400], dtype=torch.int32, device=dev), torch.tensor([430, 100], dtype=torch.int32, device=dev)
w = torch.zeros(2, 2, 448, device=dev)
call = lambda: (K.attn_paged(q, k, v, t, cu, lens, 0.1, 300, 430, weights=w, weights_out=w.clone()), K.kv_evict_paged(k.clone(), v.clone(), w + 1, t, lens, nt, 60, 4))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a, b = call()
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    c, d = call()
    assert all(torch.equal(x, y) for x, y in zip(a + b, c + d))
print('equal')
"""


def test_first_call_inside_a_capture():
    """a process whose first calls are captured: the kernels' attributes are set there"""
    r = subprocess.run([sys.executable, '-c', FIRST_CALL], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and 'equal' in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize('new', [1, 80, 300])
def test_absent_pages_of_long_tables(dev, K, new):
    """more than 64 pages per sample, one of the last ones missing; and a sample that has all of them beside it"""
    run_attention(K, dev, [new, new], [3000, 1500], 2, 1, 64, 16, weights=True, absent=[(0, 100, -1), (0, 187, 10 ** 8)])
    run_attention(K, dev, [new, new], [3000, 2100], 2, 2, 128, 32, absent=[(1, 65, -5)])


@pytest.mark.parametrize('H,hk', [(32, 1), (40, 2), (17, 1)])
def test_many_heads_per_kv_head(dev, K, H, hk):
    """single tokens whose group alone is more than the rows of the form for few"""
    run_attention(K, dev, [1, 1], [300, 70], H, hk, 64, 32, weights=True, packed=True)
    run_attention(K, dev, [3, 1], [90, 513], H, hk, 128, 16, weights=True)


def test_long_lists_of_row_tiles(dev, K):
    """more than a thousand row tiles: whole caches one after the other"""
    run_attention(K, dev, [80, 70, 80, 66, 80], [80, 100, 90, 70, 85], 16 * 48, 48, 32, 16, packed=True)


@pytest.mark.parametrize('new', [20, 200])
@pytest.mark.parametrize('hd', [32, 128])
def test_the_largest_probability_is_not_rounded(dev, K, new, hd):
    """a key in every later 64-key tile scores a little (0.4 to 4.9 log2 units) more than all before it, and only the last one has values in
    the first column: there the result is v / sum with one rounding, the result's own (2^-8), if the subtracted maximum is the maximum"""
    g = torch.Generator().manual_seed(new + hd)
    H, L = 4, 64 * 6
    k = torch.zeros(6, H, 64, hd)
    v = torch.randn(6, H, 64, hd, generator=g).bfloat16()
    v[:, :, :, 0] = 0
    step = torch.rand(6, H, generator=g) * 4.5 + 0.4
    height = step.cumsum(0)
    k[:, :, 5, 0] = height.bfloat16().float()                                # token 5 of a tile stands out
    v[5, :, 5, 0] = 1 + torch.rand(H, generator=g).bfloat16()
    q = torch.zeros(new, H, hd)
    q[:, :, 0] = 1 + torch.rand(new, H, generator=g) / 16                    # every row another sum
    k, q = k.bfloat16(), q.view(new, H * hd).bfloat16()
    table, scale = torch.arange(6, dtype=torch.int32)[None], 0.6931471805599453
    rest = R.attention(q, k, v, table, [new], [L], scale)
    out, _ = K.attn_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), i32([0, new], dev), i32([L], dev), scale, new, L)
    got, want = out.cpu().double().view(new, H, hd)[..., 0], rest[0].view(new, H, hd)[..., 0]
    seen = torch.arange(L - new, L) >= 5 * 64 + 5                            # the rows that see the last one that stands out
    assert (got[~seen] == 0).all()
    # numerator: exactly v; sum and quotient in fp32 (scores: one product, base and scale rounded), then one rounding
    tol = want.abs() * (R.U_BF16 + (L + 64) * R.U_F32)
    assert ((got - want).abs() <= tol)[seen].all(), float(((got - want).abs() / want.abs())[seen].max() / R.U_BF16)


def test_append_of_rows_without_a_sample(dev, K):
    """a table of no sample: nothing is stored, the rows' q is rotated all the same"""
    g = torch.Generator().manual_seed(2)
    H, hk, hd, T = 4, 2, 64, 5
    k = torch.full((4, hk, 16, hd), 2.0, dtype=torch.bfloat16, device=dev)
    v, table = k.clone(), torch.zeros(0, 3, dtype=torch.int32)
    qkv = torch.randn(T, (H + 2 * hk) * hd, generator=g).bfloat16()
    ang = torch.rand(8, hd, generator=g) * 6
    seq, idx, pos = torch.zeros(T, dtype=torch.int32), torch.arange(T, dtype=torch.int32), torch.arange(1, T + 1, dtype=torch.int32)
    want = R.append(qkv, seq, idx, table, k.cpu(), v.cpu(), pos, ang.cos(), ang.sin(), H)
    q = torch.full((T, H * hd), 5.0, dtype=torch.bfloat16, device=dev)
    K.kv_append_paged(qkv.to(dev), seq.to(dev), idx.to(dev), table.to(dev), k, v, pos.to(dev), ang.cos().to(dev), ang.sin().to(dev), H, q_out=q)
    close(q, want[0], want[1])
    assert (k == 2).all() and (v == 2).all()


@pytest.mark.parametrize('budget', [64, 200])
def test_who_is_not_over_the_budget_keeps_its_pages(dev, K, budget):
    """the new table names the old pages of a sample all of whose tokens stay: its rows, weights and indices are what they were"""
    g = torch.Generator().manual_seed(budget)
    lens, hk, hd, page = [50, 700, budget, 0], 2, 64, 16
    k, v, tab = R.make_cache(lens + [budget], hk, hd, page, g)
    table, new_table = tab[:4], tab[:4].clone()
    new_table[1] = tab[4]
    w = torch.rand(4, hk, 720, generator=g)
    kept, new = R.evict(w, table, k.shape[0], page, lens, budget, 8)
    kd, vd = k.to(dev), v.to(dev)
    nw, nl, got = K.kv_evict_paged(kd, vd, w.to(dev), table.to(dev), i32(lens, dev), new_table.to(dev), budget, 8)
    assert nl.tolist() == new == [50, budget, budget, 0]
    ke, ve = k.clone(), v.clone()
    at = torch.arange(budget)
    for h in range(hk):
        for b in range(4):
            assert got[b, h].tolist() == kept[b][h] + [-1] * (budget - new[b])
            assert torch.equal(nw[b, h].cpu()[:new[b]], w[b, h][kept[b][h]]) and (nw[b, h, new[b]:] == 0).all()
        idx = torch.tensor(kept[1][h])
        src, dst = table[1].long()[idx // page], new_table[1].long()[at // page]
        ke[dst, h, at % page], ve[dst, h, at % page] = k[src, h, idx % page], v[src, h, idx % page]
    assert torch.equal(kd.cpu().view(torch.int16), ke.view(torch.int16)) and torch.equal(vd.cpu().view(torch.int16), ve.view(torch.int16))


def test_cache_evicts_a_ragged_batch(dev):
    """one sample over the budget, one under it: free pages are needed for the first only, the second stays where it is"""
    from mmmm_amd.models.cogvlm.kv_cache import PagedKVCache
    c = PagedKVCache(2, 2, 256, 2, 64, dev, page_size=16, n_pages=16, track_weights=True)
    lens = [180, 20]                                         # 12 + 2 pages: two are free
    c.begin(torch.cat([torch.zeros(180), torch.ones(20)]).to(dev), torch.cat([torch.arange(180), torch.arange(20)]).to(dev), i32(lens, dev), 180)
    c.commit()
    assert c.lens.tolist() == lens and c.free_pages == 2 and c.len_bounds == lens
    c.k.normal_()
    c.v.normal_()
    c.weights[:, 0, :, :180].uniform_()
    c.weights[:, 1, :, :20].uniform_()
    rows = lambda x, b, idx: torch.stack([x[c.block_table[b].long()[j // 16], :, j % 16] for j in idx], 1)      # noqa: E731  [heads, tokens, hd]
    old = [[[rows(x[layer], b, range(n)) for x in (c.k, c.v)] for b, n in enumerate(lens)] for layer in range(2)]
    w, table = c.weights.clone(), c.block_table.cpu().clone()
    c.evict(24, 4)
    assert c.lens.tolist() == [24, 20] == c.len_bounds and c.free_pages == 12 and torch.equal(c.block_table[1].cpu(), table[1])
    assert torch.equal(c.weights[:, 1], w[:, 1])
    for layer in range(2):
        kept, _ = R.evict(w[layer].cpu(), table, 16, 16, lens, 24, 4)
        for b in range(2):
            for n, x in enumerate((c.k, c.v)):
                now = rows(x[layer], b, range(c.lens.tolist()[b]))
                for h in range(2):
                    assert torch.equal(now[h], old[layer][b][n][h][kept[b][h]])
                    assert torch.equal(c.weights[layer, b, h, :len(kept[b][h])], w[layer, b, h][kept[b][h]])


@pytest.mark.parametrize('budget,recent', [(100, 10), (33001, 5000), (39999, 0)])
@pytest.mark.parametrize('kind', ['random', 'ties'])
def test_evict_of_more_tokens_than_lds_holds_keys(dev, K, budget, recent, kind):
    """beyond 32768 tokens the keys are made again in every pass; the shorter sample beside it keeps its keys in LDS"""
    g = torch.Generator().manual_seed(budget)
    lens, hk, hd, page = [40000, 700], 2, 32, 256
    k, v, tab = R.make_cache(lens + [min(n, budget) for n in lens], hk, hd, page, g)
    table, new_table = tab[:2], tab[2:]
    table[0, 1] = -1                                                         # 256 tokens that are not there
    w = torch.rand(2, hk, 40000, generator=g)
    if kind == 'ties':
        w = (w * 50).floor()
    kept, new = R.evict(w, table, k.shape[0], page, lens, budget, recent)
    kd, vd = k.to(dev), v.to(dev)
    nw, nl, got = K.kv_evict_paged(kd, vd, w.to(dev), table.to(dev), i32(lens, dev), new_table.to(dev), budget, recent)
    assert nl.tolist() == new
    ke, ve = k.clone(), v.clone()
    for b in range(2):
        for h in range(hk):
            idx = torch.tensor(kept[b][h])
            n = len(idx)
            assert torch.equal(got[b, h, :n].cpu().long(), idx) and (got[b, h, n:] == -1).all()
            assert torch.equal(nw[b, h, :n].cpu(), w[b, h][idx]) and (nw[b, h, n:] == 0).all()
            at = torch.arange(n)
            src, dst = table[b].long()[idx // page], new_table[b].long()[at // page]
            ke[dst, h, at % page], ve[dst, h, at % page] = k[src, h, idx % page], v[src, h, idx % page]
    assert torch.equal(kd.cpu().view(torch.int16), ke.view(torch.int16)) and torch.equal(vd.cpu().view(torch.int16), ve.view(torch.int16))


FIRST_EVICTION = """
import torch
from mmmm_amd import kernels as K
dev = torch.device('cuda', 0)
g = torch.Generator().manual_seed(0)
k, v = (torch.randn(20, 2, 64, 128, generator=g).bfloat16().to(dev) for _ in range(2))
t = torch.arange(14, dtype=torch.int32, device=dev).view(2, 7)
nt = torch.tensor([[15, 17, 18], [14, 16, -1]], dtype=torch.int32, device=dev)     # pages that nothing else uses
lens = torch.tensor([430, 100], dtype=torch.int32, device=dev)
w = torch.rand(2, 2, 448, generator=g).to(dev)
torch.cuda.synchronize()
for budget in (60, 129):                                  # rows moved by the select itself; by a launch of their own
    k1, v1 = k.clone(), v.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = K.kv_evict_paged(k1, v1, w, t, lens, nt, budget, 4)
    for _ in range(3):
        k1.copy_(k)
        v1.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        k2, v2 = k.clone(), v.clone()
        b = K.kv_evict_paged(k2, v2, w, t, lens, nt, budget, 4)
        assert all(torch.equal(x, y) for x, y in zip(a + (k1, v1), b + (k2, v2)))
    for s in range(2):
        for h in range(2):
            for j, i in enumerate(a[2][s, h].tolist()):
                if i >= 0:
                    assert torch.equal(k1[int(nt[s, j // 64]), h, j % 64], k[int(t[s, i // 64]), h, i % 64])
                    assert torch.equal(v1[int(nt[s, j // 64]), h, j % 64], v[int(t[s, i // 64]), h, i % 64])
    assert torch.equal(k1[:14], k[:14]) and torch.equal(v1[:14], v[:14])
print('equal')
"""


def test_first_eviction_inside_a_capture_moves_the_rows():
    """a process whose first call is a captured eviction, into pages of its own: indices, weights and the moved rows on every replay"""
    r = subprocess.run([sys.executable, '-c', FIRST_EVICTION], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and 'equal' in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize('new,L', [(1, 3000), (3, 100), (40, 2500), (300, 700)])
def test_output_over_the_queries(dev, K, new, L):
    """out=q without weights: the same bits; with weights it is refused"""
    args, kw = _case(K, dev, new, L, 7, weights=True)
    want, lse = K.attn_paged(*args)
    q = args[0].clone()
    got, lse2 = K.attn_paged(q, *args[1:], out=q)
    assert got is q and torch.equal(got, want) and torch.equal(lse, lse2)
    with pytest.raises(AssertionError):
        K.attn_paged(q, *args[1:], out=q, **kw)


@pytest.mark.parametrize('new', [[1, 1, 1], [3, 0, 1], [40, 1, 20], [300, 30, 1]])
@pytest.mark.parametrize('H,hk,hd', [(4, 2, 128), (3, 3, 64)])
def test_bounds_far_above_the_lengths(dev, K, new, H, hk, hd):
    """what a step captured once for the whole table passes: max_q and max_kv of tables and chunks far longer than what is there"""
    g = torch.Generator().manual_seed(sum(new))
    lens, page, cols, rows = [700, 33, 260], 32, 400, 2000
    k, v, table = R.make_cache(lens, hk, hd, page, g, cols=cols)
    T = sum(new)
    q = torch.randn(rows, H * hd, generator=g).bfloat16()
    w = torch.rand(3, hk, cols * page, generator=g)
    want = R.attention(q, k, v, table, new, lens, hd ** -0.5, None, w)
    cu = [0, new[0], new[0] + new[1], T]
    wo = torch.full_like(w, -1.0).to(dev)
    out = torch.full((rows, H * hd), 3.0, dtype=torch.bfloat16, device=dev)
    _, lse = K.attn_paged(q.to(dev), k.to(dev), v.to(dev), table.to(dev), i32(cu, dev), i32(lens, dev), hd ** -0.5, rows, cols * page, weights=w.to(dev),
                          weights_out=wo, out=out)
    close(out[:T], want[0][:T], want[1][:T], 'out')
    close(lse[:, :T], want[2][:, :T], want[3][:, :T], 'lse')
    assert (out[T:] == 3.0).all()
    for b, L in enumerate(lens):
        close(wo[b, :, :L], want[4][b, :, :L], want[5][b, :, :L], 'weights')
        assert (wo[b, :, L:] == -1.0).all()
