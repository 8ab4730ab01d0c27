"""Refusals of the paged-cache entry points: everything a host can see is checked before a launch (no GPU needed)."""
import ctypes as C

import pytest
import torch

from mmmm_amd import hip, kernels as K

BAD, UNSUPPORTED, OK = -1, -2, 0
P = 1 << 20                       # an aligned address that is never followed: every call below ends before a launch


@pytest.fixture(scope='module')
def lib():
    from mmmm_amd import build
    build.build(verbose=False)
    return hip.lib()


def cache(**kw):
    c = hip.PagedKVArgs()
    d = dict(k_pages=P, v_pages=P, ld_page=2 * 64 * 128, n_pages=4, page_size=64, block_table=P, ld_table=3, max_pages=3, n_seq=2, n_kv_heads=2, head_dim=128)
    d.update(kw)
    for k, v in d.items():
        setattr(c, k, v)
    return c


CACHE_BAD = [(dict(k_pages=None), BAD), (dict(v_pages=None), BAD), (dict(block_table=None), BAD), (dict(n_pages=0), BAD), (dict(max_pages=0), BAD),
             (dict(n_kv_heads=0), BAD), (dict(n_seq=-1), BAD), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
             (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(page_size=2048, ld_page=1 << 20), UNSUPPORTED),
             (dict(k_pages=P + 8), BAD), (dict(ld_page=2 * 64 * 128 - 8), BAD), (dict(ld_page=2 * 64 * 128 + 4), BAD), (dict(ld_table=2), BAD),
             (dict(max_pages=1 << 26, ld_table=1 << 26), UNSUPPORTED)]


def attn(c=None, **kw):
    a = hip.AttnPagedArgs()
    a.cache = c or cache()
    d = dict(q=P, ldq=512, cu_q=P, kv_lens=P, row_of_pos=None, out=P, ldo=512, lse=P, ld_lse=10, n_rows=10, max_q=5, max_kv=100, n_heads=4, scale=0.1,
             w_cols=0, weights=None, weights_out=None)
    d.update(kw)
    for k, v in d.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('i', range(len(CACHE_BAD)))
def test_cache_refused_everywhere(lib, i):
    kw, rc = CACHE_BAD[i]
    c = cache(**kw)
    n = C.c_int64(0)
    a = attn(c)
    assert lib.vm_attn_paged_bf16(C.addressof(a), None) == rc
    assert lib.vm_attn_paged_workspace(C.addressof(a), C.addressof(n)) == rc
    assert lib.vm_kv_append_paged_bf16(C.addressof(c), P, 1024, P, P, P, P, P, 10, 4, 4, P, 512, None, None) == rc
    assert lib.vm_kv_evict_paged_bf16(C.addressof(c), P, 200, 100, 100, P, 2 * P, 3, 3, 64, 8, 2 * P, 200, 100, 2 * P, P, None) == rc


@pytest.mark.parametrize('kw,rc', [
    (dict(n_heads=3), BAD), (dict(n_heads=0), BAD), (dict(ldq=504), BAD), (dict(ldq=516), BAD), (dict(ldo=508), BAD), (dict(q=P + 2), BAD), (dict(out=P + 8), BAD),
    (dict(q=None), BAD), (dict(out=None), BAD), (dict(lse=None), BAD), (dict(ld_lse=9), BAD), (dict(cu_q=None), BAD), (dict(kv_lens=None), BAD),
    (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float('nan')), BAD), (dict(scale=float('inf')), BAD), (dict(max_q=-1), BAD), (dict(max_kv=-1), BAD),
    (dict(n_rows=-1), BAD), (dict(weights_out=P), BAD), (dict(weights=P, weights_out=P, w_cols=0), BAD),
    (dict(weights=P, weights_out=P, w_cols=100, ldw_head=99, ldwo_head=100), BAD), (dict(weights=P, weights_out=P, w_cols=100, ldw_head=100, ldwo_head=99), BAD),
])
def test_attention_refused(lib, kw, rc):
    a = attn(**kw)
    assert lib.vm_attn_paged_bf16(C.addressof(a), None) == rc


def test_attention_without_its_workspace_is_refused(lib):
    a = attn(cache(max_pages=200, ld_table=200, n_pages=4), max_q=1, max_kv=12000)
    n = C.c_int64(0)
    assert lib.vm_attn_paged_workspace(C.addressof(a), C.addressof(n)) == OK
    if n.value:
        assert lib.vm_attn_paged_bf16(C.addressof(a), None) == BAD
        a.workspace, a.workspace_bytes = P, n.value - 1
        assert lib.vm_attn_paged_bf16(C.addressof(a), None) == BAD


def test_append_refused(lib):
    good = [P, 1024, P, P, P, P, P, 10, 4, 4, P, 512, None, None]      # qkv, ld, row_seq, row_index, row_pos, cos, sin, n_pos, rows, n_heads, q_out, ldq

    def call(**kw):
        names = ['qkv', 'ld', 'row_seq', 'row_index', 'row_pos', 'cos', 'sin', 'n_pos', 'rows', 'n_heads', 'q_out', 'ldq', 'nrows', 'stream']
        args = [kw.get(n, g) for n, g in zip(names, good)]
        c = cache()
        return lib.vm_kv_append_paged_bf16(C.addressof(c), *args)
    for kw in (dict(qkv=None), dict(qkv=P + 2), dict(ld=1016), dict(ld=1028), dict(row_seq=None), dict(row_index=None), dict(row_pos=None), dict(cos=None),
               dict(sin=None), dict(sin=P + 4), dict(n_pos=0), dict(rows=-1), dict(n_heads=0), dict(q_out=None), dict(ldq=504)):
        assert call(**kw) == BAD, kw
    assert call(rows=0) == OK


def test_evict_refused(lib):
    names = ['weights', 'ldw_seq', 'ldw_head', 'w_cols', 'lens', 'new_table', 'ld_new', 'new_pages', 'budget', 'recent', 'new_w', 'ldn_seq', 'ldn_head', 'new_lens', 'kept']
    good = [P, 200, 100, 100, P, 2 * P, 3, 3, 64, 8, 2 * P, 200, 100, 2 * P, P]
    for kw in (dict(weights=None), dict(ldw_head=99), dict(w_cols=0), dict(lens=None), dict(new_table=None), dict(ld_new=2), dict(new_pages=0), dict(budget=0),
               dict(recent=-1), dict(recent=65), dict(new_w=None), dict(ldn_head=99), dict(new_lens=None), dict(kept=None), dict(new_w=P), dict(new_lens=P), dict(new_table=P), dict(new_pages=1, budget=65)):
        c = cache()
        assert lib.vm_kv_evict_paged_bf16(C.addressof(c), *[kw.get(n, g) for n, g in zip(names, good)], None) == BAD, kw


def test_struct_layouts(lib):
    assert C.sizeof(hip.PagedKVArgs) == 64 and hip.PagedKVArgs.block_table.offset == 32 and hip.PagedKVArgs.head_dim.offset == 60
    assert C.sizeof(hip.AttnPagedArgs) == 224 and hip.AttnPagedArgs.n_rows.offset == 136 and hip.AttnPagedArgs.weights.offset == 160
    assert hip.PAGED_KV.size == 64 and hip.ATTN_PAGED.size == 224
    a = attn(weights=3, weights_out=4, w_cols=5, ldw_seq=6, workspace=7, workspace_bytes=8, row_of_pos=9)
    flat = [getattr(a.cache, n) for n, _ in hip.PagedKVArgs._fields_] + [getattr(a, n) for n, _ in hip.AttnPagedArgs._fields_[1:]]
    assert hip.ATTN_PAGED.pack(*[0 if v is None else v for v in flat]) == bytes(a)


def test_wrappers_refuse_what_they_can_see():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    t = torch.zeros(2, 3, dtype=torch.int32)
    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16)
    cu, lens = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    ok = dict(q=q, k=k, v=k.clone(), t=t, cu=cu, lens=lens, scale=0.1)

    def call(**kw):
        d = {**ok, **kw}
        return K.attn_paged(d['q'], d['k'], d['v'], d['t'], d['cu'], d['lens'], d['scale'], 3, 40)
    for kw in (dict(q=q.float()), dict(q=q[:, :200]), dict(k=k.float(), v=k.float()), dict(v=k[:3]), dict(k=k.transpose(1, 2), v=k.transpose(1, 2)),
               dict(t=t.long()), dict(scale=0.0), dict(scale=float('nan')), dict(k=k[..., :48].contiguous(), v=k[..., :48].contiguous()),
               dict(k=k[:, :, :12].contiguous(), v=k[:, :, :12].contiguous())):
        with pytest.raises(AssertionError):
            call(**kw)
    with pytest.raises(hip.HipError):                      # host tensors: there is no CPU path
        call()


def test_no_sample_needs_no_table(lib):
    c = cache(n_seq=0, block_table=None)
    a = attn(c, n_rows=0, q=None, out=None, lse=None, cu_q=None, kv_lens=None)
    n = C.c_int64(-1)
    assert lib.vm_attn_paged_workspace(C.addressof(a), C.addressof(n)) == OK and n.value == 0
    assert lib.vm_attn_paged_bf16(C.addressof(a), None) == OK
    assert lib.vm_kv_append_paged_bf16(C.addressof(c), None, 1024, None, None, None, None, None, 10, 0, 4, None, 512, None, None) == OK
    assert lib.vm_kv_evict_paged_bf16(C.addressof(c), None, 200, 100, 100, None, None, 3, 3, 64, 8, None, 200, 100, None, None, None) == OK


def test_weights_out_of_one_sample_for_all_is_refused():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    w = torch.zeros(1, 2, 48)
    cu, lens = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        K.attn_paged(torch.zeros(3, 256, dtype=torch.bfloat16), k, k.clone(), torch.zeros(2, 3, dtype=torch.int32), cu, lens, 0.1, 3, 40, weights=w.expand(2, 2, 48))


@pytest.mark.parametrize('kw,want', [
    (dict(max_q=1, max_kv=12000), 2 * 2 * 2 * 24 * (128 + 4) * 4),                        # few rows: 24 key splits of 512 tokens, 2 rows per cache
    (dict(max_q=1, max_kv=12000, w_cols=12800), 2 * 2 * 2 * (24 * (128 + 4) + 12000) * 4),        # ... and their scores
    (dict(max_q=1, max_kv=400), 0),
    (dict(max_q=10, max_kv=12000), 2 * 2 * 20 * 24 * (128 + 4) * 4),                      # many rows: 24 splits again
])
def test_the_workspace_is_asked_for_and_missed(lib, kw, want):
    """what the plan needs, and the call without it, or with a byte less, or misaligned, refused"""
    if 'w_cols' in kw:
        kw = dict(kw, weights=P, weights_out=P, ldw_head=12800, ldwo_head=12800)
    a = attn(cache(max_pages=200, ld_table=200, n_pages=4), **kw)
    n = C.c_int64(-1)
    assert lib.vm_attn_paged_workspace(C.addressof(a), C.addressof(n)) == OK and n.value == want
    if want:
        assert lib.vm_attn_paged_bf16(C.addressof(a), None) == BAD
        a.workspace, a.workspace_bytes = P, want - 1
        assert lib.vm_attn_paged_bf16(C.addressof(a), None) == BAD
        a.workspace, a.workspace_bytes = P + 8, want
        assert lib.vm_attn_paged_bf16(C.addressof(a), None) == BAD


def test_weights_with_the_output_over_the_queries_are_refused(lib):
    kw = dict(weights=2 * P, weights_out=2 * P, w_cols=192, ldw_head=192, ldwo_head=192, workspace=P, workspace_bytes=1 << 40)
    a = attn(**kw)
    assert lib.vm_attn_paged_bf16(C.addressof(a), None) == BAD
