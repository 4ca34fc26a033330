"""The paged cache without a GPU: refusals of the operators, the C entry points' checks,
and PagedCache's bookkeeping (pages shared, copied, freed, compacted) against a plain
record of what each sequence holds, with the device operators replaced by torch ones."""
import ctypes
import os
import random

import pytest
import torch

import lucid_b200 as lb
from lucid_b200 import _lib, paged


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from lucid_b200 import build
        build.build()
    return _lib.load()


def test_operators_refuse_cpu_tensors():
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    tab, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: lb.paged_decode_step(q, q, q, pool, pool, tab, n, 0.1),
                 lambda: lb.paged_decode_attention(q, pool, pool, tab, n, 0.1),
                 lambda: lb.paged_append(q, q, pool, pool, tab, n),
                 lambda: lb.copy_pages(pool, pool, [0], [1]),
                 lambda: lb.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


P = ctypes.c_void_p(4096)      # an aligned address that is never followed
ODD = ctypes.c_void_p(4098)


def _step(lib, B=2, Hq=8, Hkv=2, D=64, pages=9, ps=16, M=4, q=P, k=P, kp=P, snp=64, ws=P, nws=1 << 30, tab=P):
    return lib.lucid_paged_decode_step(B, Hq, Hkv, D, pages, ps, M, 0.1, 1e-5, q, 512, 64, k, 128, 64, P, 128, 64,
                                       kp, 2048, 1024, snp, P, 2048, 1024, 64, tab, M, P, P, 128, 64, P, 512, 64, 1,
                                       None, ws, nws, None)


def test_step_argument_errors(lib):
    shape = dict(B=(-1,), Hq=(7, -8), Hkv=(0,), D=(0, 2, 66, 132), pages=(0,), ps=(0,), M=(0, 1 << 28))
    for name, values in shape.items():
        for v in values:
            assert _step(lib, **{name: v}) == 1, (name, v)
    assert _step(lib, B=0) == 0 and _step(lib, Hq=0) == 0
    assert _step(lib, q=ODD) == 2 and _step(lib, kp=ODD) == 2 and _step(lib, k=ODD) == 2
    assert _step(lib, snp=66) == 2 and _step(lib, tab=None) == 2 and _step(lib, kp=None) == 2
    need = lib.lucid_paged_decode_workspace_bytes(2, 8, 2, 64, 1)
    assert _step(lib, nws=need - 1) == 3 and _step(lib, ws=None) == 3 and _step(lib, ws=ODD) == 3


def test_workspace_holds_every_segment(lib):
    """A segment is one CTA's share of one (sequence, kv head, row block): at most CTAs +
    items of them, each of rows x (D + 4) floats; the step has one more row."""
    w = lambda *a: lib.lucid_paged_decode_workspace_bytes(*a) - 256
    one = w(1, 4, 4, 64, 0)
    assert (w(2, 4, 4, 64, 0) - one) == 4 * 1 * 68 * 4             # 4 more items of 1 row
    assert (w(2, 4, 4, 64, 1) - w(1, 4, 4, 64, 1)) == 4 * 2 * 68 * 4
    assert (w(2, 96, 4, 64, 0) - w(1, 96, 4, 64, 0)) == 4 * 2 * 12 * 68 * 4   # 24 heads: 2 blocks of 12
    assert (w(2, 64, 4, 64, 1) - w(1, 64, 4, 64, 1)) == 4 * 2 * 9 * 68 * 4    # 16 heads: 2 blocks of 8, and one


def test_append_argument_errors(lib):
    def call(B=2, H=2, N=3, D=64, pages=9, ps=16, M=4, k=P, kn=64, tab=P):
        return lib.lucid_paged_append(B, H, N, D, pages, ps, M, k, 384, 192, kn, P, 384, 192, 64, P, 2048, 1024, 64,
                                      P, 2048, 1024, 64, tab, M, P, None, None, None)
    for kw in (dict(B=-1), dict(B=65536), dict(N=-1), dict(D=66), dict(D=132), dict(pages=0), dict(ps=0), dict(M=0)):
        assert call(**kw) == 1, kw
    assert call(B=0) == 0 and call(N=0) == 0 and call(H=0) == 0
    assert call(k=ODD) == 2 and call(kn=65) == 2 and call(tab=None) == 2


def test_copy_pages_argument_errors(lib):
    """Everything a copy could do wrong is seen on the host."""
    def call(src, dst, layers=2, pages=10, size=4096, kp=P, step=4096):
        c = lambda v: (ctypes.c_int * max(1, len(v)))(*v)
        return lib.lucid_copy_pages(layers, pages, size, kp, 40960, step, P, 40960, 4096, c(src), c(dst), len(src), None)
    assert call([], []) == 0 and call([1], [2], layers=0) == 0
    for src, dst in (([1], [10]), ([10], [1]), ([-1], [1]), ([1], [-1]),
                     ([1, 2], [3, 3]),          # written twice
                     ([1, 2], [2, 3]), ([1, 2], [3, 1]), ([4], [4])):   # read and written
        assert call(src, dst) == 1, (src, dst)
    assert call([1], [2], size=0) == 1 and call([1], [2], size=4) == 1 and call([1], [2], layers=-1) == 1
    assert call([1], [2], size=1 << 40, layers=1000) == 1
    assert call([1], [2], kp=ODD) == 2 and call([1], [2], step=4098) == 2
    bad = lib.lucid_copy_pages(1, 10, 4096, P, 0, 4096, P, 0, 4096, None, None, 1, None)
    assert bad == 1


def test_token_logprobs_argument_errors(lib):
    def fwd(R0=1, R1=4, V=100, dtype=0, x=P, top=2, tokens=P, lp=P, ent=P, tv=P):
        return lib.lucid_token_logprobs(R0, R1, V, dtype, x, 0, V, tokens, top, lp, ent, P, tv, P, None, None)
    for kw in (dict(V=0), dict(dtype=3), dict(dtype=-1), dict(top=65), dict(top=-1), dict(V=1), dict(R0=-1),
               dict(R0=1 << 20, R1=1 << 20)):
        assert fwd(**kw) == 1, kw
    assert fwd(R0=0) == 0 and fwd(R1=0) == 0
    odd = ctypes.c_void_p(4097)
    assert fwd(x=odd) == 2 and fwd(x=ODD, dtype=2) == 2 and fwd(lp=None) == 2 and fwd(ent=None) == 2 and fwd(tv=None) == 2
    bwd = lambda V=100, x=P, d=P: lib.lucid_token_logprobs_bwd(1, 4, V, 0, x, 0, 100, P, P, P, P, d, None)
    assert bwd(V=0) == 1 and bwd(x=odd) == 2 and bwd(d=None) == 2


def test_rows_past_the_index_range_are_refused(lib):
    """An element index runs past a row's end by a batch of vectors, within 32 bits."""
    for V in ((1 << 30) + 1, (1 << 31) - 65):
        assert lib.lucid_token_logprobs(1, 1, V, 0, P, 0, V, None, 0, None, P, None, None, None, None, None) == 1
        assert lib.lucid_token_logprobs_bwd(1, 1, V, 0, P, 0, V, None, P, P, P, P, None) == 1


def test_rows_of_logits_as_two_strided_dimensions():
    from lucid_b200.logprobs import _row_view
    x = torch.zeros(4, 3, 5, 8)
    assert _row_view(x)[1:] == (1, 60, 0, 8)
    assert _row_view(x[:, :, :-1])[1:] == (12, 4, 40, 8)
    assert _row_view(x[:, :2, :-1])[1:] == (1, 32, 0, 8)                    # three strides: copied
    assert _row_view(x[0, 0, 0])[1:3] == (1, 1)
    assert _row_view(x[:1].expand(4, 3, 5, 8))[1:] == (4, 15, 0, 8)
    for empty in (x[:, :, :0], torch.zeros(0, 3, 2, 8).transpose(0, 2), x[:0]):
        assert 0 in _row_view(empty)[1:3]                                   # and it returns


def test_status_words_name_their_cause():
    assert _lib.decode_status(4 | (16 << 20)).startswith("paged decoding: a page of the block table")
    assert _lib.decode_status(5 | (17 << 20)).startswith("paged append: a length or a new row lies past")
    assert _lib.decode_status(6 | (18 << 20)).startswith("token log probabilities: a token lies outside")


def test_page_numbers():
    assert list(paged._ids([1, 2], "src")) == [1, 2] and list(paged._ids(torch.tensor([3, 4]), "src")) == [3, 4]
    for bad in ([1.5], ["a"], [1 << 40], torch.tensor([1.0]), torch.tensor([[1]]), torch.tensor([True])):
        with pytest.raises(TypeError):
            paged._ids(bad, "src")


# ---------------------------------------------------------------------------
# bookkeeping
# ---------------------------------------------------------------------------
def _plain_copy(key_pages, x_pages, src, dst):
    src, dst = list(src), list(dst)
    assert len(set(dst)) == len(dst) and not set(src) & set(dst)
    for pool in (key_pages, x_pages):
        pool[:, dst] = pool[:, src].clone()


def _plain_append(key, x, key_pages, x_pages, table, lengths, counts):
    ps = key_pages.shape[2]
    for b in range(key.shape[0]):
        for i in range(int(counts[b])):
            t = int(lengths[b]) + i
            page = int(table[b, t // ps])
            key_pages[page, :, t % ps] = key[b, :, i]
            x_pages[page, :, t % ps] = x[b, :, i]


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(paged, "copy_pages", _plain_copy)
    monkeypatch.setattr(paged, "paged_append", _plain_append)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def _cache(pages=12, ps=4):
    return lb.PagedCache(2, 1, 4, pages, ps, device="cpu")


def _held(cache, seq, layer):
    """The first element of every cached key row of a sequence."""
    n = cache.length(seq)
    rows = [cache.key_pages[layer, p, 0, :, 0] for p in cache.pages(seq)]
    return torch.cat(rows)[:n].tolist() if rows else []


def _write(batch, counts, values, layers=2):
    batch.reserve(counts)
    n = max(counts)
    k = torch.zeros(len(batch), 1, n, 4, dtype=torch.bfloat16)
    for b, row in enumerate(values):
        k[b, 0, :len(row), 0] = torch.tensor(row, dtype=torch.bfloat16)
    for layer in range(layers):
        batch.append(layer, k + layer, k)
    batch.advance()


def test_cache_bookkeeping_against_a_plain_record(on_cpu):
    """Random appends, forks, frees and compactions; every sequence keeps its own tokens
    and every page is either free or referenced as often as lists name it."""
    rng, cache, record, value = random.Random(7), _cache(pages=40), {}, 0
    for step in range(400):
        act = rng.random()
        if act < 0.15 or not record:
            for s in cache.new(rng.randint(1, 2)):
                record[s] = []
        elif act < 0.25:
            s = rng.choice(sorted(record))
            record[cache.fork(s)] = list(record[s])
        elif act < 0.35:
            s = rng.choice(sorted(record))
            cache.free(s)
            del record[s]
        elif act < 0.42:
            before = cache.free_pages
            cache.compact()
            used = {p for s in record for p in cache._sequences[s].pages}
            assert cache.free_pages == before and used == set(range(len(used)))
        else:
            seqs = rng.sample(sorted(record), rng.randint(1, len(record)))
            counts = [rng.randint(0, 6) for _ in seqs]
            batch, free, refs = cache.batch(seqs), cache.free_pages, list(cache._refs)
            rows = [[float((value + i) % 250) for i in range(n)] for n in counts]
            try:
                _write(batch, counts, rows) if max(counts) else batch.reserve(counts)
            except lb._lib.LucidError as e:
                assert "is full" in str(e) and cache.free_pages == free and cache._refs == refs
                for s in seqs[:2]:
                    cache.free(s)
                    del record[s]
                continue
            if max(counts):
                for s, row in zip(seqs, rows):
                    record[s] += row
            value += 7
        named = [p for s in record for p in cache._sequences[s].pages]
        assert [named.count(p) for p in range(40)] == cache._refs
        assert sorted(cache._free) == [p for p in range(40) if cache._refs[p] == 0]
        for s in record:
            assert cache.length(s) == len(record[s])
            for layer in range(2):
                assert _held(cache, s, layer) == [v + layer for v in record[s]], (step, s)


def test_full_cache_changes_nothing(on_cpu):
    cache = _cache(pages=3)
    a, b = cache.new(2)
    _write(cache.batch([a]), [6], [[1, 2, 3, 4, 5, 6]])          # two pages
    child = cache.fork(a)
    batch = cache.batch([a, child, b])
    refs, free = list(cache._refs), cache.free_pages
    with pytest.raises(_lib.LucidError, match="2 pages needed, 1 of 3 free"):
        batch.reserve([1, 0, 1])                                  # a copy for a, a page for b
    assert cache._refs == refs and cache.free_pages == free and cache.pages(a) == cache.pages(child)
    batch.reserve([1, 0, 0])                                      # a alone: its shared page is copied
    assert cache.pages(a)[0] == cache.pages(child)[0] and cache.pages(a)[1] != cache.pages(child)[1]


def test_both_forks_writing_copies_once(on_cpu):
    cache = _cache()
    a, = cache.new()
    _write(cache.batch([a]), [2], [[1, 2]])
    c = cache.fork(a)
    free = cache.free_pages
    _write(cache.batch([a, c]), [1, 1], [[3], [4]])
    assert cache.free_pages == free - 1 and _held(cache, a, 0) == [1, 2, 3] and _held(cache, c, 0) == [1, 2, 4]


def test_reserve_again_and_stale_batches(on_cpu):
    cache = _cache()
    a, b = cache.new(2)
    batch = cache.batch([a, b])
    k = torch.zeros(2, 1, 3, 4, dtype=torch.bfloat16)
    with pytest.raises(_lib.LucidError, match="reserve"):
        batch.append(0, k, k)
    batch.reserve(3)
    free = cache.free_pages
    batch.reserve([3, 2])                                         # the pages are already there
    assert cache.free_pages == free
    with pytest.raises(ValueError, match="3 tokens were reserved"):
        batch.append(0, k[:, :, :2], k[:, :, :2])
    with pytest.raises(ValueError, match="one token"):
        batch.step(0, k, k, k, 0.1)
    cache.fork(a)                                                 # pages may be shared now
    for call in (lambda: batch.append(0, k, k), batch.advance):
        with pytest.raises(_lib.LucidError, match="reserve again"):
            call()
    batch.reserve([3, 2])
    batch.advance()
    assert batch.host_lengths == [3, 2] and batch.lengths.tolist() == [3, 2] and batch.get_seq_length() == 3
    cache.free(b)
    with pytest.raises(_lib.LucidError, match="not in the cache"):
        batch.reserve(1)


def test_two_batches_with_the_same_sequence(on_cpu):
    """The one that advances first wins; the other would write over its rows."""
    cache = _cache()
    a, b, c = cache.new(3)
    one, two, other = cache.batch([a, b]), cache.batch([b]), cache.batch([c])
    k = torch.zeros(2, 1, 1, 4, dtype=torch.bfloat16)
    for batch in (one, two, other):
        batch.reserve(1)
    two.append(0, k[:1], k[:1])
    two.advance()
    for call in (lambda: one.append(0, k, k), one.advance):
        with pytest.raises(_lib.LucidError, match="another batch"):
            call()
    other.append(0, k[:1], k[:1])                                 # shares nothing with it
    other.advance()
    one.reserve(1)
    one.advance()
    assert [cache.length(s) for s in (a, b, c)] == [1, 2, 1]


def test_a_failing_page_copy_changes_nothing(on_cpu, monkeypatch):
    """copy_pages also raises what an earlier call reported."""
    cache = _cache()
    a, = cache.new()
    _write(cache.batch([a]), [2], [[1, 2]])
    child = cache.fork(a)
    refs, free, batch = list(cache._refs), cache.free_pages, cache.batch([child])

    def fails(*args):
        raise _lib.LucidError("reported before")
    with monkeypatch.context() as m:
        m.setattr(paged, "copy_pages", fails)
        with pytest.raises(_lib.LucidError, match="reported before"):
            batch.reserve(3)
    assert cache._refs == refs and cache.free_pages == free and cache.pages(a) == cache.pages(child)
    with pytest.raises(_lib.LucidError, match="reserve"):
        batch.advance()
    _write(batch, [1], [[3]])
    assert _held(cache, child, 0) == [1, 2, 3] and _held(cache, a, 0) == [1, 2]


def test_bookkeeping_stays_out_of_captures(on_cpu, monkeypatch):
    cache = _cache()
    batch = cache.batch(cache.new())
    batch.reserve(1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: batch.reserve(1), batch.advance, cache.compact):
        with pytest.raises(_lib.LucidError, match="works on the host"):
            call()
    assert batch.host_lengths == [0]


def test_refusals_of_the_cache(on_cpu):
    cache = _cache()
    a, = cache.new()
    for bad in ([], [a, a]):
        with pytest.raises(ValueError):
            cache.batch(bad)
    with pytest.raises(_lib.LucidError):
        cache.batch([a + 1])
    with pytest.raises(_lib.LucidError):
        cache.free(99)
    for bad in ([1, 1], [-1], -1):
        with pytest.raises(ValueError):
            cache.batch([a]).reserve(bad)
    for kw in (dict(head_dim=66), dict(head_dim=132), dict(num_pages=0), dict(page_size=0), dict(num_layers=0)):
        with pytest.raises(ValueError):
            lb.PagedCache(**{**dict(num_layers=1, num_kv_heads=1, head_dim=64, num_pages=2, page_size=4, device="cpu"), **kw})


def test_decoder_refuses_what_a_paged_cache_cannot_take(on_cpu):
    from lucid_b200.decoder import LucidForCausalLM, lucid_config
    cfg = lucid_config(hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=4,
                       num_key_value_heads=2, head_dim=16, vocab_size=50)
    model = LucidForCausalLM(cfg).init_weights().eval()
    cache = lb.PagedCache.for_config(cfg, 8, 4, device="cpu")
    batch = cache.batch(cache.new(2))
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="PagedBatch"):
        model(ids, prompt_lengths=[1, 2])
    for bad in ([1], [0, 2], [1, 4]):
        with pytest.raises(ValueError, match="do not fit"):
            model(ids, batch, prompt_lengths=bad)
    with pytest.raises(ValueError, match="logits_to_keep"):
        model(ids, batch, prompt_lengths=[1, 2], logits_to_keep=2)
    with pytest.raises(ValueError, match="3 rows of ids"):
        model(torch.zeros(3, 3, dtype=torch.int64), batch)
    with pytest.raises(ValueError, match="two tokens"):
        model.score(ids[:, :1])
    with pytest.raises(ValueError, match="max_new_tokens"):
        model.generate(ids, batch, 0)
    with pytest.raises(RuntimeError, match="eval"):
        model.train()(ids, batch)
    model.eval()
    batch.reserve([2, 0])
    batch.advance()
    with pytest.raises(NotImplementedError, match="begun"):
        model(ids[:, :1], batch)
    batch.reserve([1, 1])
    batch.advance()
    with pytest.raises(NotImplementedError, match="3 tokens"):
        model(ids, batch)


# ---------------------------------------------------------------------------
# the dealing out of tiles (csrc/paged_decode.cu), in plain integers
# ---------------------------------------------------------------------------
TILE, COST = 64, 2


def _segments(lens, per, nctas):
    """(cta, item, first tile, tiles) of every segment, as the tile pass walks its units."""
    tiles = [-(-n // TILE) for n in lens]
    units = [(t + COST if t else 0) for t in tiles]
    T = sum(units) * per
    G, out = min(T, nctas), []
    for cta in range(G):
        at, left = cta * T // G, (cta + 1) * T // G - cta * T // G
        b = 0
        while at >= units[b] * per:
            at -= units[b] * per
            b += 1
        hb, tile = at // units[b], at % units[b] - COST
        while left > 0:
            skip = max(0, min(-tile, left))
            tile, left = tile + skip, left - skip
            if left == 0:
                break
            n = min(tiles[b] - tile, left)
            out.append((cta, b * per + hb, tile, n))
            left, tile = left - n, tile + n
            if tile == tiles[b] and left > 0:
                tile, hb = -COST, hb + 1
                if hb == per:
                    hb, b = 0, b + 1
                    while tiles[b] == 0:
                        b += 1
    return out, T, G


def test_tiles_are_dealt_out_once_and_joined_where_they_went():
    """Every tile of every item in exactly one segment; an item's segments are those of the
    CTAs that the join computes, all of them, in order; slots cta + item are never shared
    and stay inside the workspace."""
    rng = random.Random(3)
    for trial in range(300):
        B, per, nctas = rng.randint(1, 40), rng.choice([1, 2, 4, 6, 32]), rng.choice([1, 7, 148, 444])
        lens = [rng.choice([0, 1, 63, 64, 65, rng.randint(1, 300), rng.randint(1, 20000)]) for _ in range(B)]
        got, T, G = _segments(lens, per, nctas)
        slots = [cta + item for cta, item, _, _ in got]
        assert len(set(slots)) == len(slots) and max(slots, default=0) < nctas + B * per
        by_item = {}
        for cta, item, tile, n in got:
            assert n > 0
            by_item.setdefault(item, []).append((cta, tile, n))
        before = 0
        for b, n in enumerate(lens):
            nt = -(-n // TILE)
            for hb in range(per):
                mine = by_item.get(b * per + hb, [])
                if nt == 0:
                    assert not mine
                    continue
                first = before + hb * (nt + COST) + COST
                i0, i1 = ((first + 1) * G - 1) // T, ((first + nt) * G - 1) // T
                assert [c for c, _, _ in mine] == list(range(i0, i1 + 1)), (lens, per, nctas)
                at = 0
                for _, tile, k in mine:
                    assert tile == at
                    at += k
                assert at == nt
            before += (nt + COST) * per if nt else 0
