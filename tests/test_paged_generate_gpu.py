"""The generation path over a paged cache: the same tokens and logits as over the contiguous one, conversations that go on, finished samples,
captured steps, eviction by received weight. bf16 bounds as in test_generate_gpu.py (two bf16 evaluations of the same logits)."""
import pytest
import torch

from tests._gpu_common import rel
from tests.test_generate_gpu import _forced, _sample
from tests.test_model_gpu import lm, make_inputs  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu


def _batch(batch):
    vi = batch['vlm_inputs']
    return vi['input_ids'], dict(token_type_ids=vi['token_type_ids'], position_ids=vi['position_ids'], attention_mask=vi['attention_mask'],
                                 image=batch['image'], patch_size=batch['patch_size'], pool_size=batch['pool_size'])


@pytest.mark.parametrize('page', [16, 64])
def test_paged_equals_contiguous(dev, lm, page):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    forced = _forced(tok, 6, 3, 5).to(dev)
    a = lm.generate(ids, **kw, forced_tokens=forced, return_logits=True)
    b = lm.generate(ids, **kw, forced_tokens=forced, return_logits=True, kv_page_size=page)
    assert torch.equal(a.new_position_ids, b.new_position_ids) and torch.equal(a.past_key_values.lens, b.past_key_values.lens)
    for t in range(6):
        assert rel(b.logits[t], a.logits[t]) < 1e-2, t
    # what is cached is the same rows, in other places
    ca, cb = a.past_key_values, b.past_key_values
    H, hd = cb.n_heads, cb.head_dim
    for s in range(3):
        n = int(ca.lens[s])
        j = torch.arange(n, device=dev)
        rows = cb.k[0][cb.block_table[s].long()[j // page], :, j % page]
        assert rel(rows.reshape(n, H * hd).float(), ca.k[0, s, :n].float()) < 1e-2


def test_conversation_goes_on(dev, lm):
    """second turn: a chunk of further tokens over the filled cache gives the logits of one full forward over everything"""
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    kw, img = _sample(batch, 2)
    n = kw['input_ids'].shape[1]
    f1, f2 = _forced(tok, 4, 1, 3).to(dev), _forced(tok, 5, 1, 4).to(dev)
    g = torch.Generator().manual_seed(9)
    question = torch.randint(3, 150, (1, 7), generator=g).to(dev)
    cache = lm.new_kv_cache(1, n + 40, dev, page_size=16)                 # room for both turns
    one = lm.generate(**kw, **img, forced_tokens=f1, return_logits=True, past_key_values=cache)
    assert one.past_key_values is cache
    chunk = torch.cat([f1[:, -1:], question], 1)
    last = one.new_position_ids[:, -1:]
    pos = torch.cat([last, last + 1 + torch.arange(7, device=dev)], 1)
    two = lm.generate(chunk, token_type_ids=torch.zeros_like(chunk), position_ids=pos, image=None, patch_size=None, pool_size=None,
                      forced_tokens=f2, return_logits=True, past_key_values=cache)
    ids = torch.cat([kw['input_ids'], f1, question, f2[:, :-1]], 1)
    tt = torch.cat([kw['token_type_ids'], torch.zeros(1, ids.shape[1] - n, dtype=torch.long, device=dev)], 1)
    allpos = torch.cat([kw['position_ids'], one.new_position_ids, pos[:, 1:], two.new_position_ids[:, :-1]], 1)
    lm.eval()
    with torch.no_grad():
        full = lm(ids, token_type_ids=tt, position_ids=allpos, **img)
    at = n + f1.shape[1] + 7 - 1
    for t in range(5):
        assert rel(two.logits[t][0], full.logits[0, at + t]) < 2e-2, t
    assert two.past_key_values.lens.tolist() == [ids.shape[1]]


def test_single_token_turn(dev, lm):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    kw, img = _sample(batch, 0)
    f = _forced(tok, 6, 1, 7).to(dev)
    whole = lm.generate(**kw, **img, forced_tokens=f, return_logits=True, kv_page_size=16)
    cache = lm.new_kv_cache(1, kw['input_ids'].shape[1] + 10, dev, page_size=16)
    first = lm.generate(**kw, **img, forced_tokens=f[:, :3], return_logits=True, past_key_values=cache)
    rest = lm.generate(f[:, 2:3], token_type_ids=torch.zeros_like(f[:, :1]), position_ids=first.new_position_ids[:, -1:], image=None, patch_size=None,
                       pool_size=None, forced_tokens=f[:, 3:], return_logits=True, past_key_values=cache)
    for t in range(3):
        assert rel(rest.logits[t], whole.logits[3 + t]) < 1e-2
    assert torch.equal(rest.past_key_values.lens, whole.past_key_values.lens)


def test_graph_replayed_paged_decode_equals_eager(dev, lm):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    for extra in ({}, dict(kv_budget=24, kv_recent=8)):
        eager = lm.generate(ids, **kw, max_new_tokens=40, kv_page_size=16, **extra)
        graphed = lm.generate(ids, **kw, max_new_tokens=40, kv_page_size=16, use_graph=True, **extra)
        assert torch.equal(eager.new_tokens, graphed.new_tokens) and torch.equal(eager.new_position_ids, graphed.new_position_ids)
        assert graphed.past_key_values.lens.tolist() == eager.past_key_values.lens.tolist()


def test_finished_samples_store_nothing(dev, lm):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    free = lm.generate(ids, **kw, max_new_tokens=12, kv_page_size=16)
    eos = int(free.new_tokens[0, 3])
    n = kw['attention_mask'].sum(1).tolist()
    for graph in (False, True):
        out = lm.generate(ids, **kw, max_new_tokens=12, kv_page_size=16, eos_token_id=eos, eos_check_every=100, use_graph=graph)
        for s in range(3):
            toks = out.new_tokens[s].tolist()
            fed = toks.index(eos) if eos in toks[:-1] else len(toks) - 1        # the eos itself, and what follows it, is not cached
            assert int(out.past_key_values.lens[s]) == n[s] + fed, (graph, s)


def test_budget(dev, lm):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    longest = int(kw['attention_mask'].sum(1).max())
    forced = _forced(tok, 40, 3, 6).to(dev)
    want = lm.generate(ids, **kw, forced_tokens=forced, return_logits=True, kv_page_size=16)
    wide = lm.generate(ids, **kw, forced_tokens=forced, return_logits=True, kv_page_size=16, kv_budget=longest + 100, kv_recent=8)
    assert all(torch.equal(a, b) for a, b in zip(want.logits, wide.logits))             # nothing left: the same bits
    w = wide.past_key_values.weights
    total = w.sum((1, 2, 3)) if w.dim() == 4 else None
    fed = wide.past_key_values.lens.sum().item() * wide.past_key_values.n_heads          # every query gives one in all per head
    assert torch.allclose(total.cpu(), torch.full_like(total.cpu(), fed), rtol=1e-4)
    cut = lm.generate(ids, **kw, forced_tokens=forced, return_logits=True, kv_page_size=16, kv_budget=24, kv_recent=8)
    c = cut.past_key_values
    assert int(c.lens.max()) < 24 + 16 and c.max_len < want.past_key_values.max_len + 16
    assert all(torch.isfinite(x).all() for x in cut.logits)
    assert torch.equal(cut.logits[0], want.logits[0])                                    # the prompt itself saw everything
    with pytest.raises(ValueError):
        lm.generate(ids, **kw, max_new_tokens=4, kv_budget=24)
    with pytest.raises(ValueError):
        lm.generate(ids, **kw, max_new_tokens=4, kv_page_size=16, kv_budget=24, kv_recent=25)
    with pytest.raises(ValueError):
        lm.generate(ids, **kw, max_new_tokens=4, past_key_values=lm.new_kv_cache(3, 200, dev))
    with pytest.raises(ValueError):
        lm.generate(ids, **kw, max_new_tokens=4, past_key_values=want.past_key_values, kv_budget=24)


@pytest.mark.parametrize('graph', [False, True])
@pytest.mark.parametrize('width', [1, 6])
def test_a_sample_sits_a_turn_out(dev, lm, width, graph):
    """one sample has nothing to say in the second turn: nothing of it is stored, the others answer as they would without it"""
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    g = torch.Generator().manual_seed(3)
    said = torch.randint(3, 150, (3, width), generator=g).to(dev)
    answers = []
    for silent in (None, 1):
        cache = lm.new_kv_cache(3, ids.shape[1] + 40, dev, page_size=16)
        one = lm.generate(ids, **kw, max_new_tokens=3, past_key_values=cache)
        before = cache.lens.tolist()
        mask = torch.ones_like(said)
        if silent is not None:
            mask[silent] = 0
        pos = one.new_position_ids[:, -1:] + torch.arange(width, device=dev)
        two = lm.generate(said, token_type_ids=torch.zeros_like(said), position_ids=pos, attention_mask=mask, image=None, patch_size=None, pool_size=None,
                          max_new_tokens=6, past_key_values=cache, use_graph=graph)
        assert cache.lens.tolist() == [n if s == silent else n + width + 5 for s, n in enumerate(before)]
        answers.append(two.new_tokens)
    assert torch.equal(answers[0][[0, 2]], answers[1][[0, 2]])


def test_live_flags_belong_to_a_paged_cache(dev, lm):
    ids, pos = torch.zeros(2, dtype=torch.long, device=dev), torch.zeros(2, dtype=torch.long, device=dev)
    live = torch.ones(2, dtype=torch.bool, device=dev)
    with pytest.raises(AssertionError):
        lm.model.decode_step(ids, pos, lm.new_kv_cache(2, 32, dev), live)
    with pytest.raises(AssertionError):
        lm.model.decode_step(ids, pos, lm.new_kv_cache(2, 32, dev, page_size=16), live[:1])


@pytest.mark.parametrize('graph', [False, True])
def test_a_silent_sample_of_the_first_call_stores_nothing(dev, lm, graph):
    """a cache made by the call itself, no eos: a sample without a valid token is not cached, and the conversation goes on without it"""
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(3, 150, (3, 9), generator=g).to(dev)
    mask = torch.ones_like(ids)
    mask[1] = 0
    mask[2, 6:] = 0
    kw = dict(token_type_ids=torch.zeros_like(ids), position_ids=torch.arange(9, device=dev).expand(3, 9).contiguous(), image=None, patch_size=None, pool_size=None)
    out = lm.generate(ids, attention_mask=mask, **kw, max_new_tokens=6, kv_page_size=16, use_graph=graph)
    assert out.past_key_values.lens.tolist() == [9 + 5, 0, 6 + 5]
    alone = lm.generate(ids[:1], **{k: v[:1] if v is not None else None for k, v in kw.items()}, max_new_tokens=6, kv_page_size=16, use_graph=graph)
    assert torch.equal(out.new_tokens[:1], alone.new_tokens)


@pytest.mark.parametrize('graph', [False, True])
def test_a_ragged_batch_in_a_pool_that_just_holds_it(dev, lm, graph):
    """pages for the tokens there are, not for batch x longest: the same tokens as in a pool with room for all, one page less is refused"""
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    g = torch.Generator().manual_seed(6)
    lens, steps, page = [90, 7, 30], 20, 16
    ids = torch.randint(3, 150, (3, 90), generator=g).to(dev)
    mask = (torch.arange(90)[None] < torch.tensor(lens)[:, None]).long().to(dev)
    kw = dict(token_type_ids=torch.zeros_like(ids), position_ids=torch.arange(90, device=dev).expand(3, 90).contiguous(), attention_mask=mask,
              image=None, patch_size=None, pool_size=None, max_new_tokens=steps, use_graph=graph)
    want = lm.generate(ids, **kw, kv_page_size=page)
    need = sum(-(-(n + steps - 1) // page) for n in lens)
    assert need < want.past_key_values.k.shape[1] * 2 // 3
    cache = lm.new_kv_cache(3, 90 + steps, dev, page_size=page, n_pages=need)
    out = lm.generate(ids, **kw, past_key_values=cache)
    assert torch.equal(out.new_tokens, want.new_tokens) and cache.lens.tolist() == [n + steps - 1 for n in lens] and cache.launch_new is None
    small = lm.new_kv_cache(3, 90 + steps, dev, page_size=page, n_pages=need - 1)
    with pytest.raises(ValueError, match='overflow'):
        lm.generate(ids, **kw, past_key_values=small)
    assert small.launch_new is None


@pytest.mark.parametrize('graph', [False, True])
def test_a_finished_sample_takes_no_pages(dev, lm, graph):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    g = torch.Generator().manual_seed(8)
    ids = torch.randint(3, 150, (2, 14), generator=g).to(dev)
    kw = dict(token_type_ids=torch.zeros_like(ids), position_ids=torch.arange(14, device=dev).expand(2, 14).contiguous(), image=None, patch_size=None,
              pool_size=None, max_new_tokens=40, use_graph=graph)
    free = lm.generate(ids, **kw, kv_page_size=16)
    first = [int(free.new_tokens[0, 0]), int(free.new_tokens[1, 0])]
    s = 0 if first[0] not in free.new_tokens[1].tolist() else 1 if first[1] not in free.new_tokens[0].tolist() else None
    if s is None:
        pytest.skip('both samples say the same')
    cache = lm.new_kv_cache(2, 14 + 40, dev, page_size=16, n_pages=1 + 4)    # 14 tokens of the one that ends at once, 53 of the other
    out = lm.generate(ids, **kw, past_key_values=cache, eos_token_id=first[s], eos_check_every=100)
    assert cache.lens.tolist()[s] == 14 and cache.lens.tolist()[1 - s] == 53
    assert torch.equal(out.new_tokens[1 - s], free.new_tokens[1 - s])


class _Stop(Exception):
    pass


def _fails_after(f, good):
    """f, whose call number `good` (from 0) raises"""
    def call(*args):
        nonlocal good
        good -= 1
        if good < 0:
            raise _Stop
        return f(*args)
    return call


@pytest.mark.parametrize('graph', [False, True])
def test_a_failed_turn_leaves_the_conversation_as_it_was(dev, lm, graph, monkeypatch):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    g = torch.Generator().manual_seed(4)
    said = torch.randint(3, 150, (3, 5), generator=g).to(dev)
    answers = []
    for failing in (False, True):
        cache = lm.new_kv_cache(3, ids.shape[1] + 40, dev, page_size=16)
        one = lm.generate(ids, **kw, max_new_tokens=3, past_key_values=cache)
        turn = dict(token_type_ids=torch.zeros_like(said), position_ids=one.new_position_ids[:, -1:] + torch.arange(5, device=dev), patch_size=None, pool_size=None,
                    max_new_tokens=6, past_key_values=cache, use_graph=graph)
        if failing:
            before = cache.lens.tolist()
            with pytest.raises(AssertionError):
                lm.generate(said, **{**turn, 'image': batch['image'][:1], 'patch_size': batch['patch_size'][:1], 'pool_size': batch['pool_size'][:1]})
            layers = len(lm.model.layers)
            for calls in (0, 1, 2):                          # in the last layer of the chunk; of the first step; of the next (the captured one)
                with monkeypatch.context() as m:
                    m.setattr(type(cache), 'attend', _fails_after(type(cache).attend, calls * layers + layers - 1))
                    with pytest.raises(_Stop):
                        lm.generate(said, **turn, image=None)
                assert cache.launch_bound is None and cache.launch_new is None
                assert cache.tighten() == [n + (0, 5, 6)[calls] for n in before]
                cache.lens.copy_(torch.tensor(before, dtype=torch.int32))      # the finished calls of the turn are taken back
                cache.tighten()
        answers.append(lm.generate(said, **turn, image=None).new_tokens)
    assert torch.equal(*answers)


def test_weights_that_count_a_failed_call_are_not_evicted_by(dev, lm, monkeypatch):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    cache = lm.new_kv_cache(3, ids.shape[1] + 200, dev, page_size=16, track_weights=True)
    with pytest.raises(AssertionError):                      # before the first layer: nothing was counted
        lm.generate(ids, **{**kw, 'image': batch['image'][:1]}, max_new_tokens=3, past_key_values=cache)
    lm.generate(ids, **kw, max_new_tokens=3, past_key_values=cache, kv_budget=24, kv_recent=8)
    assert int(cache.lens.max()) < 24 + 16
    said = ids[:, :4].clone()
    turn = dict(token_type_ids=torch.zeros_like(said), position_ids=torch.arange(4, device=dev).expand(3, 4).contiguous(), image=None, patch_size=None,
                pool_size=None, max_new_tokens=30, past_key_values=cache)
    with monkeypatch.context() as m:
        m.setattr(type(cache), 'append', _fails_after(type(cache).append, 1))
        with pytest.raises(_Stop):
            lm.generate(said, **turn)
    with pytest.raises(RuntimeError, match='received weights'):
        lm.generate(said, **turn, kv_budget=24, kv_recent=8)
    assert lm.generate(said, **turn).new_tokens.shape == (3, 30)


@pytest.mark.parametrize('graph', [False, True])
@pytest.mark.parametrize('budget', [None, 24])
def test_positions_beyond_the_configured_ones(dev, lm, monkeypatch, graph, budget):
    """a conversation that crosses max_position_embeddings, in a step and in a chunk: the same answers as where the limit is far away"""
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    top = int((kw['position_ids'] * kw['attention_mask']).max()) + 1
    g = torch.Generator().manual_seed(12)
    said = torch.randint(3, 150, (3, 9), generator=g).to(dev)
    runs = []
    for limit in (2048, top + 5):                            # crossed in the fifth step
        monkeypatch.setattr(lm.config, 'max_position_embeddings', limit)
        cache = lm.new_kv_cache(3, ids.shape[1] + 120, dev, page_size=16, track_weights=budget is not None)
        extra = dict(past_key_values=cache, use_graph=graph, **(dict(kv_budget=budget, kv_recent=8) if budget else {}))
        one = lm.generate(ids, **kw, max_new_tokens=30, **extra)
        pos = one.new_position_ids[:, -1:] + torch.arange(9, device=dev)
        two = lm.generate(said, token_type_ids=torch.zeros_like(said), position_ids=pos, image=None, patch_size=None, pool_size=None, max_new_tokens=25, **extra)
        last = lm.generate(said[:, :1], token_type_ids=torch.zeros_like(said[:, :1]), position_ids=two.new_position_ids[:, -1:] + 40, image=None,
                           patch_size=None, pool_size=None, max_new_tokens=5, **extra)
        runs.append([one, two, last, cache.k[:, cache.block_table[0, 0].long()].clone()])
    for a, b in zip(runs[0][:3], runs[1][:3]):
        assert torch.equal(a.new_tokens, b.new_tokens) and torch.equal(a.new_position_ids, b.new_position_ids)
    assert torch.equal(runs[0][3], runs[1][3])


def test_tables_do_not_grow_inside_a_capture(dev, lm, monkeypatch):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    top = int((kw['position_ids'] * kw['attention_mask']).max()) + 1
    monkeypatch.setattr(lm.config, 'max_position_embeddings', top + 1)
    cache = lm.new_kv_cache(3, ids.shape[1] + 4 * top, dev, page_size=16)
    lm.eval()
    with torch.no_grad():
        lm(ids, **kw, past_key_values=cache, use_cache=True)
        tok1, pos = ids[:, 0].contiguous(), torch.full((3,), top, device=dev)
        cache.reserve(ids.shape[1] + 3 * top)
        x = torch.zeros(4, device=dev)
        with pytest.raises(RuntimeError, match='captured'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                x.add_(1)
                lm.model.decode_step(tok1, pos, cache)
        before = cache.tighten()
        cache.reserve(ids.shape[1] + 3 * top)
        eager = lm.model.decode_step(tok1, pos, cache)       # the tables grow here
        assert cache.lens.tolist() == [n + 1 for n in before]
        cache.lens.copy_(torch.tensor(before, dtype=torch.int32))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lm.model.decode_step(tok1, pos, cache)
        for _ in range(3):
            cache.lens.copy_(torch.tensor(before, dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_a_turn_leaves_the_pages_of_a_captured_step(dev, lm):
    """pages reserved for a captured step stay through generate(): its replays store their tokens"""
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    ids, kw = _batch(batch)
    cache = lm.new_kv_cache(3, ids.shape[1] + 100, dev, page_size=16)
    lm.generate(ids, **kw, max_new_tokens=2, past_key_values=cache)
    cache.reserve(ids.shape[1] + 90)
    tok1, pos = ids[:, 0].contiguous(), torch.full((3,), 40, device=dev)
    lm.eval()
    lm.model.decode_step(tok1, pos, cache)
    bounds = cache.len_bounds
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        lm.model.decode_step(tok1, pos, cache)
    cache.len_bounds = bounds
    free = cache.free_pages
    said = ids[:, :1].clone()
    lm.generate(said, token_type_ids=torch.zeros_like(said), position_ids=pos[:, None], image=None, patch_size=None, pool_size=None, max_new_tokens=3,
                past_key_values=cache)
    assert cache.free_pages == free
    before = cache.settle()
    for _ in range(40):
        graph.replay()
    now = cache.settle()
    assert now == [n + 40 for n in before]
    assert all(int(p) >= 0 for b in range(3) for p in cache.block_table[b, :-(-now[b] // 16)])


def test_rotary_tables_are_whole_on_every_stream(dev):
    """tables that were asked for first on a busy stream are read on another one"""
    from mmmm_amd.models.cogvlm.modeling_cogvlm import RotaryEmbedding
    r = RotaryEmbedding(64).to(dev)
    r.tables(16, dev)                                        # (the kernels are loaded)
    want = RotaryEmbedding(64).to(dev).tables(4096, dev)
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(200_000_000)                       # a tenth of a second
        r.tables(4096, dev)
    with torch.cuda.stream(other):
        got = [t.clone() for t in r.tables(4096, dev)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_chunk_with_the_mask_of_the_whole_conversation(dev, lm):
    batch, tok = make_inputs(dev)
    lm.tokenizer = tok
    g = torch.Generator().manual_seed(15)
    ids, said = (torch.randint(3, 150, (2, n), generator=g).to(dev) for n in (11, 6))
    mask, now = torch.ones_like(ids), torch.ones_like(said)
    mask[1, 4:] = 0
    now[0, 5] = 0
    lm.eval()
    out = []
    with torch.no_grad():
        for m in (now, torch.cat([mask, now], 1)):
            cache = lm.new_kv_cache(2, 40, dev, page_size=16)
            lm(ids, token_type_ids=torch.zeros_like(ids), attention_mask=mask, position_ids=torch.arange(11, device=dev).expand(2, 11), past_key_values=cache, use_cache=True)
            kw = dict(token_type_ids=torch.zeros_like(said), attention_mask=m, position_ids=11 + torch.arange(6, device=dev).expand(2, 6), past_key_values=cache)
            out.append(lm(said, **kw).logits)
            assert cache.lens.tolist() == [16, 10]
        assert torch.equal(out[0][now.bool()], out[1][now.bool()])
        for bad in (dict(attention_mask=now[:, :3]), dict(position_ids=torch.arange(17, device=dev).expand(2, 17)), dict(token_type_ids=torch.zeros(2, 17, dtype=torch.long, device=dev))):
            with pytest.raises(ValueError):
                lm(said, **{**kw, **bad})
        assert cache.settle() == [16, 10]
