"""Host side of PagedKVCache: which pages a sample has, when the table is uploaded, what is refused. No kernel runs."""
import pytest
import torch

from mmmm_amd.models.cogvlm.kv_cache import PagedKVCache


def cache(**kw):
    return PagedKVCache(2, 3, 100, 4, 32, 'cpu', **{**dict(page_size=16), **kw})


def test_pages_are_handed_out_once_and_come_back():
    c = cache()
    assert c.max_len == 112 and c.free_pages == 21 and len(c) == 0
    c.reserve(33)
    used = c.block_table[:, :3].flatten().tolist()
    assert len(set(used)) == 9 and min(used) >= 0 and (c.block_table[:, 3:] == -1).all() and c.free_pages == 12
    c.reserve(20)                                            # already there
    assert c.free_pages == 12
    c.lens.copy_(torch.tensor([33, 1, 0]))
    c.len_bound = 33
    assert c.tighten() == [33, 1, 0] and c.free_pages == 17 and c.len_bound == 33
    assert (c.block_table >= 0).sum(1).tolist() == [3, 1, 0]
    c.reserve(112)
    assert c.free_pages == 0 and sorted(c.block_table.flatten().tolist()) == list(range(21))


def test_steps_count_tokens():
    c = cache()
    c.begin(torch.tensor([0, 0, 1, 2]), torch.tensor([0, 1, 0, 0]), torch.tensor([2, 1, 1]), 2)
    assert c._row_index.tolist() == [0, 1, 0, 0] and c.lens_after().tolist() == [2, 1, 1] and c.attn_bound() == 2
    c.commit()
    c.begin(torch.tensor([0, -1, 2]), torch.zeros(3, dtype=torch.int32), torch.tensor([1, 0, 1]), 1)
    assert c._row_index.tolist()[0] == 2 and c._row_seq.tolist() == [0, -1, 2]
    assert c.lens_after().tolist() == [3, 0, 2]              # the sample without a new token is left out
    c.commit()
    assert c.lens.tolist() == [3, 1, 2] and c.len_bound == 3 and len(c) == 2


def test_refusals():
    c = cache()
    with pytest.raises(ValueError):
        c.reserve(113)
    with pytest.raises(ValueError):
        cache(n_pages=5).reserve(32)
    for bad in (8, 24, 2048):
        with pytest.raises(ValueError):
            cache(page_size=bad)
    with pytest.raises(TypeError):
        cache(dtype=torch.float32)
    with pytest.raises(ValueError):
        c.evict(8, 2)                                        # nothing was tracked
    t = cache(track_weights=True)
    for budget, recent in ((0, 0), (8, 9), (8, -1)):
        with pytest.raises(ValueError):
            t.evict(budget, recent)
    t.evict(8, 2)                                            # empty: nothing to do
    t.reserve(112)
    t.len_bound = 112
    with pytest.raises(ValueError):
        t.evict(8, 2)                                        # no page is free to move to
    t.begin(t.rows, t.zeros, t.ones, 0)
    with pytest.raises(AssertionError):
        t.tighten()


def turn(c, new, most=None):
    """one call with new[b] further tokens of sample b, of which the host knows that they are at most `most`"""
    rows = [(b, i) for b, n in enumerate(new) for i in range(n)]
    seq, off = (torch.tensor(x, dtype=torch.int32) for x in zip(*rows))
    c.begin(seq, off, torch.tensor(new, dtype=torch.int32), max(new) if most is None else most)
    pages = [[int(c.block_table[b, int(j) // c.page_size]) for b, j in zip(seq.tolist(), c._row_index.tolist())]]
    assert min(pages[0]) >= 0                               # every row has its page
    c.commit()


@pytest.mark.parametrize('lens,page,n_pages', [((4000, 100), 64, 65), ((1000, 10), 16, 64), ((1, 700, 33), 16, 48)])
def test_samples_of_different_lengths_share_a_pool_that_just_holds_them(lens, page, n_pages):
    c = PagedKVCache(1, len(lens), 4096, 2, 32, 'cpu', page_size=page, n_pages=n_pages)
    turn(c, lens)
    left = [-(-n // page) * page - n for n in lens]          # room in the last pages
    for _ in range(min(left)):
        turn(c, [1] * len(lens))
    assert c.lens.tolist() == [n + min(left) for n in lens] and c.free_pages == n_pages - sum(-(-n // page) for n in lens)
    used = c.block_table[c.block_table >= 0].tolist()
    assert len(set(used)) == len(used)
    before = c.tighten()
    with pytest.raises(ValueError):                          # one more does not fit, and nothing has changed
        turn(c, [page * n_pages] * len(lens))
    assert c.lens.tolist() == before and c.tighten() == before


def test_a_short_sample_goes_on_beside_a_long_one():
    c = PagedKVCache(1, 2, 112, 2, 32, 'cpu', page_size=16)
    turn(c, [100, 10])
    turn(c, [0, 20])
    assert c.lens.tolist() == [100, 30]
    for _ in range(12):
        turn(c, [1, 1])
    turn(c, [0, 1])                                          # the long one is full
    assert c.lens.tolist() == [112, 43] and c.attn_bound is not None and c.len_bound == 112
    with pytest.raises(ValueError):
        turn(c, [1, 1])
    assert c.lens.tolist() == [112, 43]


def test_bounds_are_a_samples_own():
    c = PagedKVCache(1, 3, 256, 2, 32, 'cpu', page_size=16, n_pages=16)
    turn(c, [200, 3, 0], most=200)                           # 13 + 1 pages
    assert c.len_bounds == [200, 3, 0] and c.free_pages == 2 and c.len_bound == 200
    c.begin(torch.tensor([0, 1], dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.tensor([1, 1, 0], dtype=torch.int32), 1)
    assert c.attn_bound() == 201
    c.commit()
    c.prepare_step(torch.tensor([False, False, False]))
    assert c.launch_new == [1, 1, 1]
    c.count_step()
    assert c.len_bounds == [202, 5, 2]
    c.launch_new = None
    assert c.tighten() == [201, 4, 0] and c.len_bounds == [201, 4, 0]


def test_a_captured_steps_pages_go_to_the_samples_that_go_on():
    c = PagedKVCache(1, 2, 64, 2, 32, 'cpu', page_size=16, n_pages=3)
    turn(c, [16, 16])                                        # both at the end of a page, one page left
    with pytest.raises(ValueError):
        c.prepare_step(torch.tensor([False, False]))
    c.prepare_step(torch.tensor([True, False]))
    assert c.launch_new == [0, 1] and (c.block_table >= 0).sum(1).tolist() == [1, 2]
    c.count_step()
    assert c.len_bounds == [16, 17]


def test_reserved_pages_stay_until_tighten():
    c = PagedKVCache(1, 2, 64, 2, 32, 'cpu', page_size=16, n_pages=5)
    c.reserve(32)
    turn(c, [20, 3])
    with pytest.raises(ValueError):
        turn(c, [13, 30], most=30)                           # 3 + 3 pages
    assert (c.block_table >= 0).sum(1).tolist() == [2, 2]    # (the lengths were read; what is reserved stayed)
    turn(c, [13, 1], most=30)
    assert c.tighten() == [33, 4] and c.free_pages == 1


def test_eviction_needs_pages_for_those_over_the_budget_only():
    c = PagedKVCache(1, 3, 256, 2, 32, 'cpu', page_size=16, track_weights=True)
    c.lens.copy_(torch.tensor([200, 20, 0]))
    c.len_bounds = [200, 20, 0]
    assert c.pages_to_evict(32) == 2 and c.pages_to_evict(16) == 2 and c.pages_to_evict(200) == 0
    c.evict(200, 8)                                          # nobody is over it: nothing to do (no kernel here)
    assert c.len_bounds == [200, 20, 0]


def test_a_dropped_call():
    c = cache(track_weights=True)
    turn(c, [5, 6, 7])
    one = torch.zeros(1, dtype=torch.int32)
    c.begin(one, one, torch.tensor([1, 0, 0], dtype=torch.int32), 1)
    c.abort()
    assert c.tighten() == [5, 6, 7] and c.len_bounds == [5, 6, 7]
    turn(c, [1, 1, 1])
    assert c.tighten() == [6, 7, 8]
    c.evict(8, 2)                                            # nobody is over it, and nothing was counted by the dropped call
    c.begin(one, one, torch.tensor([1, 0, 0], dtype=torch.int32), 1)
    c._counting = True                                       # a layer has added its weights
    c.abort()
    with pytest.raises(RuntimeError, match='received weights'):
        c.evict(8, 2)
    turn(c, [1, 1, 1])                                       # the conversation itself goes on
    assert c.tighten() == [7, 8, 9]


@pytest.mark.parametrize('good', [0, 1])
def test_a_failed_eviction_gives_its_pages_back(monkeypatch, good):
    from mmmm_amd.models.cogvlm import kv_cache
    c = cache(track_weights=True)
    c.lens.copy_(torch.tensor([60, 50, 3]))
    c.len_bounds = [60, 50, 3]
    c.reserve(60)
    free, table = c.free_pages, c.block_table.clone()
    calls = []

    def evict(k, v, w, t, lens, new, budget, recent):
        if len(calls) == good:
            raise MemoryError
        calls.append(1)
        return w, lens, None
    monkeypatch.setattr(kv_cache.K, 'kv_evict_paged', evict)
    with pytest.raises(MemoryError):
        c.evict(16, 4)
    assert c.free_pages == free and torch.equal(c.block_table, table) and c.len_bounds == [60, 50, 3] and c.lens.tolist() == [60, 50, 3]
    assert len(set(c._free)) == free
    good = 2
    if calls:
        with pytest.raises(RuntimeError, match='received weights'):
            c.evict(16, 4)
    else:
        c.evict(16, 4)
        assert c.len_bounds == [16, 16, 3]


def test_rotary_tables_grow_without_changing():
    from mmmm_amd.models.cogvlm.modeling_cogvlm import RotaryEmbedding
    for dtype in (torch.float32, torch.bfloat16):
        r = RotaryEmbedding(32).to(dtype)
        short = r.tables(64, 'cpu')
        long = r.tables(256, 'cpu')
        assert all(torch.equal(a, b[:64]) for a, b in zip(short, long)) and not torch.equal(long[0][63], long[0][200])
        assert r.tables(64, 'cpu')[0] is short[0] and r.has_tables(256, 'cpu') and not r.has_tables(128, 'cpu')      # the shorter ones stay


def test_how_long_the_rotary_tables_are():
    c = cache()
    assert c.rope_len(64) == 64
    c.pos_bound = 64
    assert c.rope_len(64) == 64
    c.pos_bound = 65
    assert c.rope_len(64) == 128
    c.reserve_positions(300)
    c.reserve_positions(10)
    assert c.rope_len(64) == 512
    d = cache()
    d.pos_bound = 1000                                       # positions may be ahead of the cached tokens (eviction)
    d.len_bounds = [10, 40, 40]
    d.reserve(60)
    assert d.rope_len(1) == 2048 and d.pos_bound == 1000
    d.reserve(100)
    assert d.rope_len(1090) == 1090 and d.rope_len(1089) == 2178


def test_eviction_leaves_the_reserved_pages(monkeypatch):
    from mmmm_amd.models.cogvlm import kv_cache
    monkeypatch.setattr(kv_cache.K, 'kv_evict_paged', lambda k, v, w, t, lens, new, budget, recent: (w, lens.clamp(max=budget), None))
    c = PagedKVCache(2, 2, 128, 4, 32, 'cpu', page_size=16, track_weights=True, n_pages=16)
    c.reserve(96)
    turn(c, [90, 20])
    assert c.settle() == [90, 20] and (c.block_table >= 0).sum(1).tolist() == [6, 6] and c.free_pages == 4
    c.evict(32, 4)
    assert c.len_bounds == [32, 20] and c.lens.tolist() == [32, 20]
    assert (c.block_table >= 0).sum(1).tolist() == [6, 6] and c.free_pages == 4
    used = c.block_table[c.block_table >= 0].tolist()
    assert len(set(used)) == 12 and not set(used) & set(c._free)
    assert c.tighten() == [32, 20] and c.free_pages == 12
