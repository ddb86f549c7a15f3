"""The paged serving path where steps are refused or cut off, scales and values are extreme, and calls come in other forms than
a serving loop's: against the 64-bit oracle, as in test_gpu_paged.py."""
import math
import random

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
PAGE = 128


@pytest.fixture(scope="module")
def sp():
    import sparse_attention_b200_b200 as m
    return m


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


# ------------------------------------------------------------------ extend_pages
def _tables(rng, old, width, spare):
    used = sum(-(-o // PAGE) for o in old)
    ids = list(range(used + spare))
    rng.shuffle(ids)
    table, at = torch.full((len(old), width), -7, dtype=torch.int32), 0
    for r, o in enumerate(old):
        c = -(-o // PAGE)
        table[r, :c] = _i32(ids[at:at + c])
        at += c
    return table, _i32(ids[at:] + [0]), _i32([spare])


def _check_extend(sp, old, new, table, free, count, total_q, total_pages):
    want = ref.extend_pages(table, _i32(old), _i32(new), free, count, total_q, total_pages)
    dev = table.cuda()
    got = sp.extend_pages(dev, _i32(old).cuda(), _i32(new).cuda(), free.cuda(), count.cuda(), total_q=total_q,
                          total_pages=total_pages)
    for name in got._fields:
        assert torch.equal(getattr(got, name).cpu(), want[name]), name
    assert torch.equal(dev.cpu(), want["table"])
    return got, dev


@pytest.mark.parametrize("old,new,spare", [
    ([0, 100], [1280, 1], 5),                                          # the second stays within its page
    ([128, 100], [129, 1], 1),
    ([100, 0, 60, 128], [1, 3000, 2, 1], 3),                           # granted, refused, no need, refused by the sum
    ([100, 100, 0, 5, 0], [300, 1, 0, 100, 0], 0),                     # nothing is free
    ([0] + [64] * 700, [900] + [1] * 700, 4),                          # many threads behind the refused one
])
def test_requests_that_need_no_page_behind_refused_ones(sp, old, new, spare):
    table, free, count = _tables(random.Random(3), old, 40, spare)
    got, _ = _check_extend(sp, old, new, table, free, count, sum(new), sum(-(-(a + b) // PAGE) for a, b in zip(old, new)))
    assert 0 <= int(got.free_count) <= spare


@pytest.mark.parametrize("batch,spare", [(40, 3), (257, 20), (3000, 9), (4096, 300)])
def test_large_batches_that_find_too_few_pages(sp, batch, spare):
    rng = random.Random(batch)
    old = [rng.choice([0, 127, 128, rng.randint(0, 1500)]) for _ in range(batch)]
    new = [rng.choice([0, 1, 1, rng.randint(0, 400)]) for _ in range(batch)]
    table, free, count = _tables(rng, old, 16, spare)
    _check_extend(sp, old, new, table, free, count, sum(new) + 5, sum(-(-(a + b) // PAGE) for a, b in zip(old, new)) + 3)


@pytest.mark.parametrize("old,new,total_pages", [([500], [1], 1), ([10, 20, 300], [700, 300, 1], 4), ([0, 5], [128, 600], 0),
                                                 ([128] * 300, [1] * 300, 450)])
def test_page_offsets_stay_within_the_page_list(sp, old, new, total_pages):
    """What reads kv_indices by cu_page_offsets (the scorer) knows no other size of it. The block table gets all pages."""
    table, free, count = _tables(random.Random(5), old, 16, 400)
    got, _ = _check_extend(sp, old, new, table, free, count, sum(new), total_pages)
    assert int(got.status) == sp.paged.STATUS_PAGES
    offsets = got.cu_page_offsets.cpu()
    assert (offsets[1:] >= offsets[:-1]).all() and int(offsets[-1]) == total_pages == got.kv_indices.numel()


def test_pages_are_neither_lost_nor_made_over_many_steps(sp):
    rng = random.Random(9)
    batch, width, pages = 300, 12, 700
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda(), _i32([pages]).cuda()
    seq = torch.zeros(batch, dtype=torch.int32, device="cuda")
    short = False
    for step in range(12):
        new = [rng.choice([0, 1, 1, 1, rng.randint(0, 300)]) for _ in range(batch)]
        b = sp.extend_pages(table, seq, _i32(new).cuda(), free, count, total_q=sum(new), total_pages=pages)
        seq, count = b.seq_lens, b.free_count
        short |= bool(int(b.status) & sp.paged.STATUS_NO_PAGES)
        held = (-(-seq.cpu().long() // PAGE)).tolist()
        assert int(count) + sum(held) == pages
        names = [p for r, h in enumerate(held) for p in table[r, :h].tolist()] + free[:int(count)].tolist()
        assert sorted(names) == list(range(pages))
    assert short


@pytest.mark.parametrize("sizes", [(2 ** 32 + 5, 3), (5, 2 ** 32 + 3), (2 ** 31, 3), (5, -2 ** 32)])
def test_extend_pages_refuses_sizes_beyond_32_bits(sp, sizes):
    one = _i32([1]).cuda()
    with pytest.raises(sp.SparseB200Error):
        sp.extend_pages(one[None].clone(), one, one, one, one, total_q=sizes[0], total_pages=sizes[1])


# ------------------------------------------------------------------ append_tokens
@pytest.mark.parametrize("old", [0.0, 2.0 ** -110, 2.0 ** -9, 0.013, 3.0])
def test_rows_behind_those_of_a_page_with_any_scale(sp, old):
    """Scales that were set elsewhere: 0 (its rows are zeros and stay so), below the lowest that is written, no power of two."""
    gen = torch.Generator().manual_seed(7)
    hkv, before, n = 2, 37, 50
    c = _cache(gen, 2, hkv)
    c["k"].view(torch.uint8)[0, :, 3, 9] = 0x7F                        # a NaN stays one
    for name in ("k_scale", "v_scale"):
        c[name][0] = old
    x = torch.randn((2, n, hkv, 128), generator=gen).to(torch.bfloat16)
    x[1] = 0                                                           # values of nothing: their scale is the lowest, or the page's
    cache = _on_gpu(sp, c)
    slots = torch.arange(before, before + n)
    sp.append_tokens(cache, x[0].cuda(), x[1].cuda(), _i32([0, n]).cuda(), slots.cuda())
    for rows, name in zip(x, ("k", "v")):
        want, want_scale = ref.append_tokens(c[name], c[name + "_scale"], rows, _i32([0, n]), slots)
        got = getattr(cache, name).cpu().double()
        assert torch.equal(getattr(cache, name + "_scale").cpu().double(), want_scale)
        assert torch.equal(got.isnan(), want.isnan())
        got, want = got.nan_to_num(0.0), want.nan_to_num(0.0)
        if math.frexp(old)[0] in (0.0, 0.5):
            assert torch.equal(got, want)
        else:                                                          # 1 / s and the product are rounded in 32 bits: a tie may fall the other way
            step = torch.exp2(torch.frexp(want)[1].clamp(min=-5).double() - 4)
            assert ((got - want).abs() <= step).all() and (got == want).double().mean() > 0.999


def test_the_tensors_of_a_cache_stay_its_own(sp):
    gen = torch.Generator().manual_seed(8)
    cache = _on_gpu(sp, _cache(gen, 3, 2))
    for name in ("k", "v", "k_scale", "v_scale", "k_index", "k_index_scale", "pages", "kv_heads", "device"):
        held = getattr(cache, name)
        with pytest.raises(sp.SparseB200Error):
            setattr(cache, name, held)
        assert getattr(cache, name) is held
    cache.layer = 3                                                    # a user's own mark
    # a tensor whose memory moves under the cache: the calls find it
    more = cache.k.clone()
    cache.k.data = more.clone()
    x = torch.randn((5, 2, 128), generator=gen).to(torch.bfloat16).cuda()
    sp.append_tokens(cache, x, x, _i32([0, 5]).cuda(), torch.arange(128, 133).cuda())
    assert not torch.equal(cache.k.view(torch.uint8)[1, :, :5], more.view(torch.uint8)[1, :, :5])
    cache.k.view(torch.uint8)[1, :, :5] = more.view(torch.uint8)[1, :, :5]
    assert torch.equal(cache.k.view(torch.uint8), more.view(torch.uint8))


# ------------------------------------------------------------------ select_pages
@pytest.mark.parametrize("pages", [12798, 12799, 12800, 51199])
def test_select_pages_of_the_longest_sequences(sp, pages):
    """Around four lists to a CTA, and the most that one list may see."""
    gen = torch.Generator(device="cuda").manual_seed(pages)
    x = torch.randn((1, pages, 3), device="cuda", generator=gen)
    got = sp.select_pages(x, _cu([3]).cuda(), _i32([pages * PAGE]).cuda(), kv_heads=1, topk=30, sink=0, recent=0, causal=False)
    assert torch.equal(got.long(), x.transpose(1, 2).topk(30, -1).indices.sort(-1).values)
    with pytest.raises(sp.SparseB200Error):
        sp.select_pages(torch.empty((1, 51200, 1), device="cuda"), _cu([1]).cuda(), _i32([5]).cuda(), kv_heads=1, topk=3)


# ------------------------------------------------------------------ paged_attention
def _cache(gen, pages, hkv):
    codes = lambda: (100 * torch.randn((pages, hkv, PAGE, 128), generator=gen)).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    scales = lambda: torch.exp2(torch.randint(-9, -5, (pages, hkv), generator=gen).float())  # noqa: E731
    return dict(k=codes(), v=codes(), k_scale=scales(), v_scale=scales())


def _on_gpu(sp, c):
    return sp.PagedCache.from_tensors(*(c[n].cuda() for n in ("k", "v", "k_scale", "v_scale")))


def _alike(sp, n, q, c, table, seq, ids=None, max_q=None, **kw):
    """out, lse (64 bits) of n requests that are all alike: [n, tokens, Hq, 128], [n, tokens, Hq]. A share then holds whole items,
    where the pages of one request alone would each be a share's own."""
    tokens, hq = q.shape[:2]
    out, lse = sp.paged_attention(q.repeat(n, 1, 1).cuda(), _on_gpu(sp, c), table.repeat(n, 1).cuda(), seq.repeat(n).cuda(),
                                  _cu([tokens] * n).cuda(), None if ids is None else ids.repeat(1, n, 1).cuda(),
                                  max_seqlen_q=tokens if max_q is None else max_q, return_lse=True, **kw)
    sp.device_status()
    return out.view(n, tokens, hq, 128).cpu().double(), lse.view(n, tokens, hq).cpu().double()


def _bounds(want, want_lse, spread, size):
    """As in test_gpu_paged.py, for queries without features far below their row's largest: a score is a sum of 128 products in
    32 bits (each addition 2^-24 of the magnitudes at most), a weight carries twice a score's error and 2^-8, an output 2^-8."""
    score = 2.0 ** -15 * size + 1e-6
    return 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * score[..., None]) * spread * 1.01 + 1e-30, score + 2.0 ** -20 * want_lse.abs()


@pytest.mark.parametrize("tokens,seq,key,order", [
    (3, 129, 127, None), (4, 130, 127, None), (4, 130, 128, None), (4, 257, 255, None), (2, 300, 299, [2, 0, 1]),
    (4, 300, 297, [2, 1, 0]),
])
@pytest.mark.parametrize("group", [1, 4])
def test_hidden_nan_values_with_further_pages_behind(sp, group, tokens, seq, key, order):
    """A NaN among the values that some tokens of an item do not see, in a page that is not the item's last: their sums are done
    again while the item goes on."""
    gen = torch.Generator().manual_seed(seq + key)
    hkv, held = 2, -(-seq // PAGE)
    c = _cache(gen, held, hkv)
    table, s = torch.randperm(held, generator=gen).to(torch.int32)[None], _i32([seq])
    q = torch.randn((tokens, hkv * group, 128), generator=gen).to(torch.bfloat16)
    bits = c["v"].view(torch.uint8)
    for d in (5, 40, 41, 127):
        bits[int(table[0, key // PAGE]), :, key % PAGE, d] = 0x7F
    # a list for all tokens: tile = tokens, whose lists are two rows apart
    tile = 1 if order is None else tokens
    ids = None if order is None else _i32(order).expand(hkv, 2, -1).contiguous()
    oracle = lambda v: ref.paged_attention(q, c["k"], v, c["k_scale"], c["v_scale"], table, s, _cu([tokens]), ids, tile)  # noqa: E731
    want, want_lse, spread, size = oracle(c["v"])
    out, lse = _alike(sp, 600, q, c, table, s, ids, tile=tile)
    assert not want[0].isnan().any() and want[-1].isnan().any()
    assert torch.equal(out.isnan(), want.isnan().expand_as(out))
    spread = oracle(torch.nan_to_num(c["v"].double(), 0.0))[2]          # of the rows that do not see it, at its features too
    bound, bound_lse = _bounds(want, want_lse, spread, size)
    assert ((out - want).abs() <= bound)[:, ~want.isnan()].all()
    assert ((lse - want_lse).abs() <= bound_lse).all()


# ------------------------------------------------------------------ the whole step
def _step(sp, lens, old, hkv, group, seed=1, index=True, wide=136):
    """A step's arguments over a fused projection whose rows are padded: q, k, v (views), cache, table, tables of the step."""
    gen = torch.Generator().manual_seed(seed)
    pages = sum(-(-(a + b) // PAGE) for a, b in zip(old, lens)) + 2
    cache = sp.PagedCache(pages, hkv, index=index)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).copy_(torch.randint(0, 0x70, t.shape, generator=gen).to(torch.uint8))
    if index:
        cache.k_index.copy_(torch.randint(0, 256, cache.k_index.shape, generator=gen).to(torch.uint8))
        cache.k_index_scale.view(torch.uint8).fill_(0x38)
    width = max(-(-(a + b) // PAGE) for a, b in zip(old, lens)) + 1
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for r, o in enumerate(old):
        table[r, :-(-o // PAGE)] = torch.arange(at, at + -(-o // PAGE))
        at += -(-o // PAGE)
    table = table.cuda()
    b = sp.extend_pages(table, _i32(old).cuda(), _i32(lens).cuda(), torch.arange(at, pages, dtype=torch.int32).cuda(),
                        _i32([pages - at]).cuda(), total_q=sum(lens), total_pages=pages)
    x = torch.randn((sum(lens), hkv * (group + 2), wide), generator=gen).to(torch.bfloat16).cuda()
    hq = hkv * group
    return x[:, :hq, :128], x[:, hq:hq + hkv, :128], x[:, hq + hkv:, :128], cache, table, b


def _copy(sp, cache):
    return sp.PagedCache.from_tensors(*(None if t is None else t.clone() for t in (
        cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_index, cache.k_index_scale)))


def _same_bits(x, y):
    return all((a is None and b is None) or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
               for a, b in zip((x.k, x.v, x.k_scale, x.v_scale, x.k_index, x.k_index_scale),
                               (y.k, y.v, y.k_scale, y.v_scale, y.k_index, y.k_index_scale)))


@pytest.mark.parametrize("topk,tile", [(None, 1), (3, 1), (3, 16)])
def test_a_step_takes_views_of_a_fused_projection(sp, topk, tile):
    q, k, v, cache, table, b = _step(sp, [20, 1, 3], [700, 900, 0], 2, 4)
    other = _copy(sp, cache)
    kw = dict(topk=topk, tile=tile, max_seqlen_q=20, max_seqlen_k=901)
    out, ids = sp.paged_step(q, k, v, cache, table, b, **kw)
    want, want_ids = sp.paged_step(q.contiguous(), k.contiguous(), v.contiguous(), other, table, b, **kw)
    assert torch.equal(out, want) and _same_bits(cache, other)
    assert (ids is None and want_ids is None) or torch.equal(ids, want_ids)
    codes, scales = sp.quantize_rows(q, 2)
    want = sp.quantize_rows(q.contiguous(), 2)
    assert torch.equal(codes, want[0]) and torch.equal(scales.view(torch.uint8), want[1].view(torch.uint8))
    for bad in (0, -2, 3, 16):
        with pytest.raises(sp.SparseB200Error):
            sp.quantize_rows(q, bad)


@pytest.mark.parametrize("bad", [
    dict(topk=0), dict(topk=3, tile=3), dict(topk=3, tile=256), dict(topk=2, sink=2, recent=1), dict(topk=2, sink=-1),
    dict(topk=2, sink=2 ** 32), dict(topk=3, max_seqlen_q=0), dict(topk=3, max_seqlen_k=0), dict(topk=3, max_seqlen_k=51200 * PAGE),
    dict(scale=math.nan), dict(scale=-math.inf), dict(topk=3, q="heads"), dict(q="strides"), dict(q="group"), dict(table="rows"),
    dict(topk=3, index=False), dict(topk=3, table="no pages"), dict(scale=1e39), dict(scale=2.0 ** 128), dict(table="wide"),
    dict(table="seq_lens"), dict(topk=3, table="cu_seqlens_k"), dict(topk=3, table="cu_page_offsets"),
    dict(topk=3, table="kv_indices"),
])
def test_a_refused_step_leaves_the_cache_as_it_was(sp, bad):
    bad = dict(bad)
    q, k, v, cache, table, b = _step(sp, [2, 1], [300, 127], 2, 4, index=bad.pop("index", True))
    q = {"heads": q[:, :3], "strides": q[..., ::2], "group": q[:, :2].repeat(1, 65, 1)}.get(bad.pop("q", None), q)
    change = bad.pop("table", None)
    if change == "rows":
        table = table[:1]
    elif change == "no pages":
        b = b._replace(kv_indices=b.kv_indices[:0])
    elif change == "wide":
        table = torch.zeros((2, 1 << 24), dtype=torch.int32, device="cuda")
    elif change == "kv_indices":
        b = b._replace(kv_indices=b.kv_indices.long())
    elif change:
        b = b._replace(**{change: getattr(b, change)[:1]})
    before = _copy(sp, cache)
    with pytest.raises(sp.SparseB200Error):
        sp.paged_step(q, k, v, cache, table, b, **{**dict(max_seqlen_q=2, max_seqlen_k=302), **bad})
    torch.cuda.synchronize()
    assert _same_bits(cache, before)


@pytest.mark.parametrize("topk,tile", [(None, 1), (3, 1), (3, 16)])
@pytest.mark.parametrize("rows", [0, 2])
def test_a_step_without_tokens(sp, topk, tile, rows):
    """No request has a new token, with and without rows of padding."""
    old, hkv = [200, 3], 2
    q, k, v, cache, table, _ = _step(sp, [1, 1], old, hkv, 4)
    b = sp.extend_pages(table, _i32(old).cuda(), _i32([0, 0]).cuda(), _i32([4]).cuda(), _i32([1]).cuda(), total_q=rows, total_pages=3)
    before = _copy(sp, cache)
    out, ids = sp.paged_step(q[:rows], k[:rows], v[:rows], cache, table, b, topk=topk, tile=tile, max_seqlen_q=1, max_seqlen_k=200)
    sp.device_status()
    assert out.shape == (rows, 8, 128) and _same_bits(cache, before)
    assert ids is None if topk is None else ids.shape == (hkv, sp.list_rows(rows, 2, tile), topk) and (ids == -1).all()


@pytest.mark.parametrize("topk", [None, 3])
def test_a_refused_request_does_not_touch_the_others(sp, topk):
    """The one in the middle finds no pages: rows and pages of the others are those of a step without it, and a step of its own
    with pages then gives what it would have given at once."""
    hkv, group, old, lens, pages = 2, 4, [300, 250, 600], [1, 200, 2], 16      # of these 3 + 2 + 5 are held, request 1 needs 2
    q, k, v, cache, table, _ = _step(sp, lens, old, hkv, group)
    grown = lambda t: torch.cat([t, t])[:pages].contiguous()  # noqa: E731
    cache = sp.PagedCache.from_tensors(*(grown(t.view(torch.uint8)).view(t.dtype) for t in (
        cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_index, cache.k_index_scale)))
    free = torch.arange(10, pages, dtype=torch.int32).cuda()

    def step(cache, table, seq, rows, lens, spare):
        b = sp.extend_pages(table, _i32(seq).cuda(), _i32(lens).cuda(), free, _i32([spare]).cuda(), total_q=sum(lens),
                            total_pages=pages)
        out, _ = sp.paged_step(q[rows], k[rows], v[rows], cache, table, b, topk=topk, max_seqlen_q=200, max_seqlen_k=602)
        return b, out

    def close(x, y, cache):
        """Another batch is cut into other shares, whose parts are joined in 32 bits: the same weights but for those of 16 bits
        (2^-11 each, relative to another reference), and each side rounds to bf16 once (2^-8 of it)."""
        most = (cache.v.float().abs() * cache.v_scale[..., None, None]).max().item()
        x, y = x.double(), y.double()
        assert ((x - y).abs() <= 2.0 ** -7 * torch.maximum(x.abs(), y.abs()) + 2.0 ** -10 * most).all()
    both, without, at_once = _copy(sp, cache), _copy(sp, cache), _copy(sp, cache)
    t1, t2, t3 = table.clone(), table.clone(), table.clone()
    b, out = step(both, t1, old, slice(0, 203), lens, 1)
    assert int(b.status) == sp.paged.STATUS_NO_PAGES and int(b.free_count) == 1 and b.seq_lens.tolist() == [301, 250, 602]
    rest = [0, 201, 202]
    assert (b.slots[1:201] == -1).all() and (b.slots[rest] >= 0).all()
    _, want = step(without, t2, old, rest, [1, 0, 2], 1)
    assert _same_bits(both, without) and torch.equal(t1, t2)
    close(out[rest], want, both)
    b, out = step(both, t1, [301, 250, 602], slice(1, 201), [0, 200, 0], 6)
    assert int(b.status) == 0 and int(b.free_count) == 4
    b, want = step(at_once, t3, old, slice(0, 203), lens, 6)
    assert _same_bits(both, at_once) and torch.equal(t1, t3)
    close(out, want[1:201], both)


# ------------------------------------------------------------------ precision of small weights and features
@pytest.mark.parametrize("depth", [4.3, 11.9, 14.4, 15.2, 16.3, 17.42, 18.6, 19.7, 20.5])
@pytest.mark.parametrize("group", [1, 4, 40])
def test_values_of_small_weights_beside_a_key_that_takes_all(sp, group, depth):
    """A key of weight 1 and value 0 (as a first token often is) in a page whose other weights are 2^-depth: the output is their
    values'. A weight is within 2^-8 of itself, or 2^-22 of the page's largest (the smallest step of its lower e4m3 term is 2^-13
    where the largest is 256, its half 2^-14)."""
    gen = torch.Generator().manual_seed(1)
    c = _cache(gen, 2, 1)
    c["k"].view(torch.uint8)[:] = 0
    c["k"][:, 0, 0, 0] = 16.0
    c["v"] = (0.5 + torch.rand(c["v"].shape, generator=gen) / 2).to(torch.float8_e4m3fn)
    c["v"][:, 0, 0] = 0.0
    c["k_scale"][:], c["v_scale"][:] = 1.0, 1.0
    q = torch.zeros((1, group, 128), dtype=torch.bfloat16)
    q[:, :, 0] = 1.0
    for seq in (128, 200, 256):
        table, s, scale = _i32([[1, 0]]), _i32([seq]), depth * math.log(2) / 16
        want, want_lse, spread, size = ref.paged_attention(q, c["k"], c["v"], c["k_scale"], c["v_scale"], table, s, _cu([1]),
                                                           scale=scale)
        bound, bound_lse = _bounds(want, want_lse, spread, size)
        # p of the page's largest is 1 / (sum of exp2 of the depths); it times 2^-22 for each of the keys' values
        weights = torch.full((seq,), 2.0 ** -depth, dtype=torch.float64)
        weights[::PAGE] = 1.0
        values = torch.cat([c["v"][1, 0], c["v"][0, 0]])[:seq].double().abs().sum(0)
        bound = bound + 2.0 ** -22 * values / weights.sum()
        out, lse = _alike(sp, 300, q, c, table, s, scale=scale)
        assert ((out - want).abs() <= bound).all(), ((out - want).abs() / bound).max()
        assert ((lse - want_lse).abs() <= bound_lse).all()


@pytest.mark.parametrize("below", [10, 14, 16, 18, 20])
@pytest.mark.parametrize("group", [1, 4, 40])
def test_scores_of_features_far_below_their_rows_largest(sp, group, below):
    """One feature of a query row, at which the keys are 0, is 2^below times the others: those make up the scores. A feature is
    off by half the smallest step of its lower e4m3 term, 2^-14 where the largest is 128 or more: 2^-21 of the largest."""
    gen = torch.Generator().manual_seed(below)
    seq = 200
    c = _cache(gen, 2, 1)
    c["k"][..., 77] = 0.0
    c["k_scale"][:] = 2.0 ** -6
    q = torch.randn((1, group, 128), generator=gen).clamp(-1.9, 1.9)
    q[:, :, 77] = 2.0 ** below * torch.linspace(1.0, 1.99, group)
    q, table, s = q.to(torch.bfloat16), _i32([[1, 0]]), _i32([seq])
    want, want_lse, spread, size = ref.paged_attention(q, c["k"], c["v"], c["k_scale"], c["v_scale"], table, s, _cu([1]))
    keys = torch.cat([c["k"][p, 0].double() * c["k_scale"][p, 0].double() for p in (1, 0)])[:seq].abs().sum(1).max()
    score = 2.0 ** -17 * size + 2.0 ** -21 * q.double().abs().amax(-1) * keys * 128 ** -0.5
    out, lse = _alike(sp, 300, q, c, table, s)
    assert ((lse - want_lse).abs() <= score + 2.0 ** -20 * want_lse.abs()).all()
    off = torch.expm1(2 * score)[..., None]
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + off) * spread * 1.01
    assert ((out - want).abs() <= bound).all(), ((out - want).abs() / bound).max()


@pytest.mark.parametrize("v_scales", [(1.0, 1e30), (1e30, 1.0), (2.0 ** 108, 2.0 ** 108), (2.0 ** -100, 2.0 ** 108)])
@pytest.mark.parametrize("rise", [0.0, 7.5, 20.0, 39.0, 45.0, 100.0])
@pytest.mark.parametrize("group", [1, 4, 40])
def test_sums_of_huge_values_stay_finite(sp, group, rise, v_scales):
    """Pages whose values are up to 2^117 and whose weights are 2^rise those of the page before: sums hold keys * largest value,
    below 2^127 here, and never a page's rise on top of it."""
    gen = torch.Generator().manual_seed(2)
    c = _cache(gen, 3, 1)
    c["k"].view(torch.uint8)[:] = 0
    c["k"][1, 0, :, 0], c["k"][2, 0, :, 0] = 8.0, 16.0                  # page 0, then 1, then 2: each rises over the one before
    c["k_scale"][:] = 1.0
    c["v_scale"][:] = torch.tensor([v_scales[0], v_scales[1], v_scales[0]])[:, None]
    q = torch.zeros((1, group, 128), dtype=torch.bfloat16)
    q[:, :, 0] = 1.0
    table, scale = _i32([[0, 1, 2]]), rise * math.log(2) / 8
    for seq in (256, 384):
        want, want_lse, spread, size = ref.paged_attention(q, c["k"], c["v"], c["k_scale"], c["v_scale"], table, _i32([seq]), _cu([1]),
                                                           scale=scale)
        bound, bound_lse = _bounds(want, want_lse, spread, size)
        # weights of 16 bits: 2^-31 of the row's largest product of weight and scale, times a code of 448, for each key
        bound = bound + seq * 448 * 2.0 ** -31 * spread.amax(-1, keepdim=True) / 100 if group > 16 else bound
        for n in (1, 600):                                             # parts of a page each, and whole items in a share
            out, lse = _alike(sp, n, q, c, table, _i32([seq]), scale=scale)
            assert out.isfinite().all()
            assert ((out - want).abs() <= bound).all(), ((out - want).abs() / bound).max()
            assert ((lse - want_lse).abs() <= bound_lse).all()


@pytest.mark.parametrize("total_pages", [0, 1, 5, 9])
def test_a_step_whose_page_list_is_cut(sp, total_pages):
    """The scorer stays within the list; requests whose pages are all in it get what they get with the whole list."""
    old, lens = [300, 250, 600], [1, 20, 2]                            # 3, 3 and 5 pages
    results = []
    for pages in (11, total_pages):
        q, k, v, cache, table, _ = _step(sp, lens, old, 2, 4)
        table[1, 2] = -1                                               # (the helper's own step has extended it)
        b = sp.extend_pages(table, _i32(old).cuda(), _i32(lens).cuda(), torch.arange(10, 13, dtype=torch.int32).cuda(),
                            _i32([3]).cuda(), total_q=23, total_pages=pages)
        if pages == 0:
            with pytest.raises(sp.SparseB200Error):                    # nothing to select from
                sp.paged_step(q, k, v, cache, table, b, topk=2, max_seqlen_q=20, max_seqlen_k=602)
            assert int(b.status) == sp.paged.STATUS_PAGES
            return
        results.append((b, *sp.paged_step(q, k, v, cache, table, b, topk=2, sink=0, max_seqlen_q=20, max_seqlen_k=602), cache))
    sp.device_status()
    (whole, out, ids, cache), (cut, out_cut, ids_cut, cache_cut) = results
    assert int(whole.status) == 0 and int(cut.status) == sp.paged.STATUS_PAGES and _same_bits(cache, cache_cut)
    assert torch.equal(whole.kv_indices[:total_pages], cut.kv_indices) and torch.equal(whole.slots, cut.slots)
    for r, end in enumerate((3, 6, 11)):
        rows = slice(int(whole.cu_seqlens_q[r]), int(whole.cu_seqlens_q[r + 1]))
        if end <= total_pages:
            assert torch.equal(ids[:, rows], ids_cut[:, rows]) and torch.equal(out[rows], out_cut[rows])
