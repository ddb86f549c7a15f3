"""The paged serving path against its 64-bit oracle: page tables, cache writer, page lists, attention over the 8-bit cache,
and the whole step. Whole numbers, codes and scales are compared exactly."""
import math
import random

import pytest
import torch

import oracle
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
def _tables(rng, old, new, width, spare, extra_stride=0):
    n = len(old)
    used = sum(min(-(-o // PAGE), width) for o in old)
    ids = list(range(used + spare))
    rng.shuffle(ids)
    table = torch.full((n, width + extra_stride), -7, dtype=torch.int32)
    at = 0
    for r, o in enumerate(old):
        c = min(-(-o // PAGE), width)
        table[r, :c] = _i32(ids[at:at + c])
        at += c
    return table, _i32(ids[at:] + [0] * 3), _i32([spare])


@pytest.mark.parametrize("old,new,width,spare,total_q,total_pages", [
    ([0], [1], 1, 1, 1, 1),
    ([127, 128, 129, 0], [1, 1, 1, 0], 4, 5, 3, 6),
    ([5, 300, 0, 1000], [128, 0, 129, 24], 9, 20, 300, 20),            # room behind the last token and page
    ([5, 300, 0, 1000], [128, 0, 129, 500], 12, 4, 757, 30),           # the last request finds too few pages
    ([100, 100, 100], [100, 28, 29], 2, 1, 157, 4),                    # pages run out in the middle, a full page still fits
    ([100, 250, 100], [300, 1, 100], 2, 9, 401, 5),                    # a row of the table is too short
    ([10, 20], [700, 300], 9, 9, 500, 4),                              # tables smaller than the step
    ([-5, 40], [3, -2], 2, 3, 3, 2),                                   # negative lengths count as nothing
    ([0, 0, 0], [0, 0, 0], 2, 2, 0, 0),
    ([0, 0], [0, 5], 2, 0, 5, 1),                                      # nothing is free
])
def test_extend_pages(sp, old, new, width, spare, total_q, total_pages):
    table, free, count = _tables(random.Random(1), old, new, width, spare, extra_stride=3)
    want = ref.extend_pages(table[:, :width], _i32(old), _i32(new), free, count, total_q, total_pages)
    dev = table.cuda()
    for _ in range(2):                                                 # the lengths are inputs: a second call gives the same
        got = sp.extend_pages(dev[:, :width], _i32(old).cuda(), _i32(new).cuda(), free.cuda(), count.cuda(), total_q=total_q,
                              total_pages=total_pages)
        for name in got._fields:
            assert torch.equal(getattr(got, name).cpu(), want[name]), name
        assert torch.equal(dev[:, :width].cpu(), want["table"])
        assert torch.equal(dev[:, width:].cpu(), table[:, width:])


@pytest.mark.parametrize("batch", [1, 31, 33, 255, 257, 1000, 4096])
def test_extend_pages_of_large_batches(sp, batch):
    rng = random.Random(batch)
    old = [rng.choice([0, 127, 128, rng.randint(0, 2000)]) for _ in range(batch)]
    new = [rng.choice([0, 1, 1, rng.randint(0, 40)]) for _ in range(batch)]
    spare = batch // 2
    table, free, count = _tables(rng, old, new, 16, spare)
    total_q, total_pages = sum(new) + 5, sum(-(-(a + b) // PAGE) for a, b in zip(old, new)) + 3
    want = ref.extend_pages(table, _i32(old), _i32(new), free, count, total_q, total_pages)
    dev = table.cuda()
    got = sp.extend_pages(dev, _i32(old).cuda(), _i32(new).cuda(), free.cuda(), count.cuda(), total_q=total_q,
                          total_pages=total_pages)
    for name in got._fields:
        assert torch.equal(getattr(got, name).cpu(), want[name]), name
    assert torch.equal(dev.cpu(), want["table"])


def test_extend_pages_of_sums_beyond_int32(sp):
    n, width = 300, 1 << 17
    old = torch.full((n,), (1 << 24) - 5, dtype=torch.int32)
    table = torch.zeros((n, width), dtype=torch.int32)
    got = sp.extend_pages(table.cuda(), old.cuda(), torch.ones_like(old).cuda(), _i32([0]).cuda(), _i32([1]).cuda(),
                          total_q=n, total_pages=4)
    assert int(got.status) & 16 and int(got.status) & 8
    assert int(got.cu_seqlens_k[-1]) == 2 ** 31 - 1 and int(got.cu_seqlens_q[-1]) == n
    assert torch.equal(got.seq_lens.cpu(), old + 1)


# ------------------------------------------------------------------ append_tokens
def _cache(gen, pages, hkv, index=True):
    codes = lambda: (100 * torch.randn((pages, hkv, PAGE, 128), generator=gen)).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    scales = lambda: torch.exp2(torch.randint(-9, -5, (pages, hkv), generator=gen).float())  # noqa: E731
    c = dict(k=codes(), v=codes(), k_scale=scales(), v_scale=scales())
    if index:
        c["k_index"] = torch.randint(256, (pages, hkv, PAGE, 64), dtype=torch.uint8, generator=gen)
        c["k_index_scale"] = torch.ones((pages, hkv, PAGE, 8)).to(torch.float8_e4m3fn)
    return c


def _on_gpu(sp, c):
    return sp.PagedCache.from_tensors(*(c[n].cuda() for n in ("k", "v", "k_scale", "v_scale")),
                                      *((c[n].cuda() for n in ("k_index", "k_index_scale")) if "k_index" in c else ()))


def _bits(t):
    return t.cpu().view(torch.uint8)


def _check_append(sp, c, k, v, cu, slots, gpu_k=None, gpu_v=None):
    cache = _on_gpu(sp, c)
    for _ in range(2):                                                 # again: the same rows at the same scales
        sp.append_tokens(cache, k.cuda() if gpu_k is None else gpu_k, v.cuda() if gpu_v is None else gpu_v, cu.cuda(),
                         slots.cuda())
    for x, codes, scale in ((k, "k", "k_scale"), (v, "v", "v_scale")):
        want, want_scale = ref.append_tokens(c[codes], c[scale], x, cu, slots)
        got = getattr(cache, codes).cpu().double()
        assert torch.equal(getattr(cache, scale).cpu().double(), want_scale)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    if "k_index" in c:
        want, want_scale = ref.append_index(c["k_index"], c["k_index_scale"], k, cu, slots)
        assert torch.equal(cache.k_index.cpu(), want) and torch.equal(_bits(cache.k_index_scale), want_scale.view(torch.uint8))


def _slots(table, old, lens):
    out = []
    for r, n in enumerate(lens):
        out += [int(table[r, p // PAGE]) * PAGE + p % PAGE for p in range(old[r], old[r] + n)]
    return torch.tensor(out, dtype=torch.int64)


@pytest.mark.parametrize("hkv,old,lens,index", [
    (1, [0], [1], True),
    (3, [5, 127, 128, 0, 250], [1, 1, 1, 128, 7], True),
    (2, [0, 64, 100], [300, 0, 29], False),
    (4, [1, 200], [500, 257], True),
])
def test_append_tokens(sp, hkv, old, lens, index):
    gen = torch.Generator().manual_seed(sum(lens))
    width = max(-(-(a + b) // PAGE) for a, b in zip(old, lens))
    pages = width * len(old) + 2
    table = torch.randperm(pages, generator=gen)[:width * len(old)].view(len(old), width)
    x = torch.randn((2, sum(lens), hkv, 128), generator=gen).to(torch.bfloat16)
    x[:, ::3] *= 0.01                                                  # runs whose scale is below their page's, and above it
    x[:, 1::7] *= 30
    _check_append(sp, _cache(gen, pages, hkv, index), x[0], x[1], _cu(lens), _slots(table, old, lens))


def test_append_tokens_from_strided_rows(sp):
    gen = torch.Generator().manual_seed(3)
    lens, hkv = [3, 130], 2
    fused = torch.randn((133, 4 + 2 * hkv, 136), generator=gen).to(torch.bfloat16)     # q heads beside k and v, padded rows
    table = torch.tensor([[4, 0], [2, 3]])
    g = fused.cuda()
    _check_append(sp, _cache(gen, 6, hkv), fused[:, 4:6, :128], fused[:, 6:8, :128], _cu(lens), _slots(table, [127, 4], lens),
                  g[:, 4:6, :128], g[:, 6:8, :128])


def test_append_tokens_special_values(sp):
    gen = torch.Generator().manual_seed(5)
    lens = [4, 2, 3, 1, 6]
    x = torch.randn((16, 1, 128), generator=gen).to(torch.bfloat16)
    x[0, 0, 3], x[1, 0, 5], x[2, 0, 7] = math.inf, -math.inf, math.nan
    x[4:6] = 0                                                         # a page of zeros: the lowest scale
    x[6:9] = 1e-38                                                     # below the lowest scale's reach
    x[9] = 3e38
    x[10:16] = torch.tensor([448.0, 449, 450, 464, 447, 896]).view(6, 1, 1).to(torch.bfloat16)
    table = torch.arange(5).view(5, 1)
    _check_append(sp, _cache(gen, 5, 1, index=False), x, x, _cu(lens), _slots(table, [0, 0, 0, 7, 0], lens))
    x[2, 0, 7] = math.inf                                              # (index vectors of NaN are not specified)
    _check_append(sp, _cache(gen, 5, 1), x, x, _cu(lens), _slots(table, [0, 0, 0, 7, 0], lens))


@pytest.mark.parametrize("top", [1e-38, 1e-3, 0.0117, 0.3, 1.0, 2.7, 6.25, 2688.0, 2700.0, 1e30])
def test_append_index_vectors_of_all_values(sp, top):
    """The conversion without a division against the rule with one: every bf16 value below `top` beside it in a group."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x[torch.isfinite(x.float()) & (x.float().abs() <= top) & (x.float().abs() >= top * 1e-5)]
    x = torch.cat([x[torch.randperm(x.numel(), generator=torch.Generator().manual_seed(1))], torch.zeros(-x.numel() % 120, dtype=x.dtype)])
    rows = torch.cat([torch.full((x.numel() // 15, 1), top).to(x.dtype), x.view(-1, 15)], 1).view(-1, 1, 128)
    n = rows.shape[0]
    cache = sp.PagedCache(-(-n // PAGE), 1)
    sp.append_tokens(cache, rows.cuda(), rows.cuda(), _i32([0, n]).cuda(), torch.arange(n).cuda())
    want, scales = oracle.quantize_nvfp4(rows)
    assert torch.equal(cache.k_index.view(-1, 64)[:n].cpu(), want[:, 0])
    assert torch.equal(_bits(cache.k_index_scale).view(-1, 8)[:n], scales.view(torch.uint8)[:, 0])


def test_append_tokens_without_a_slot_and_behind_the_last_token(sp):
    gen = torch.Generator().manual_seed(6)
    x = torch.randn((9, 1, 128), generator=gen).to(torch.bfloat16)
    slots = torch.tensor([-1, -1, 130, 131, 0, 1, 2, -1, -1], dtype=torch.int64)       # request 0 was refused, two rows of padding
    _check_append(sp, _cache(gen, 2, 1), x, x, _i32([0, 2, 4, 7]), slots)


# ------------------------------------------------------------------ select_pages
def _scores(gen, hidx, pages, cu, seq, ties):
    total = int(cu[-1]) + 3
    x = torch.randint(-3, 4, (hidx, pages, total), generator=gen).float() if ties else torch.randn((hidx, pages, total), generator=gen)
    for r in range(len(seq)):
        for t in range(int(cu[r]), int(cu[r + 1])):
            last = seq[r] - (int(cu[r + 1]) - t)
            x[:, max(0, last // PAGE + 1):, t] = -math.inf
    return x


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("lens,seq,hidx,hkv,pages,topk,tile,sink,recent", [
    ([1], [1], 1, 1, 1, 1, 1, 1, 0),
    ([1, 1, 3], [700, 5000, 1300], 4, 2, 40, 6, 1, 1, 1),
    ([5, 0, 40], [640, 10, 4000], 2, 2, 32, 9, 1, 0, 0),
    ([130, 7], [900, 2000], 3, 1, 16, 4, 64, 1, 2),
    ([130, 7, 1], [900, 2000, 129], 2, 2, 16, 5, 4, 2, 2),
    ([9], [100], 1, 1, 3, 64, 1, 1, 1),                                # a list that is longer than the sequence
    ([2, 2], [300, 40000], 1, 1, 313, 300, 1, 3, 5),
    ([4], [1], 1, 1, 2, 2, 1, 1, 1),                                   # more new tokens than keys: some see nothing
])
def test_select_pages(sp, lens, seq, hidx, hkv, pages, topk, tile, sink, recent, ties):
    gen = torch.Generator().manual_seed(len(lens) * 100 + topk)
    cu = _cu(lens)
    x = _scores(gen, hidx, pages, cu, seq, ties)
    for causal in (True, False):
        want = ref.select_pages(x, cu, seq, hkv, topk, tile, sink, recent, causal)
        got = sp.select_pages(x.cuda(), cu.cuda(), _i32(seq).cuda(), kv_heads=hkv, topk=topk, tile=tile, sink=sink, recent=recent,
                              causal=causal)
        assert torch.equal(got.cpu(), want)


def test_select_pages_of_odd_values(sp):
    cu, seq = _cu([4]), [2000]
    x = torch.full((1, 16, 4), -math.inf)
    x[0, 3, 0], x[0, 5, 0], x[0, 9, 0] = math.nan, math.inf, -1e30      # a NaN page is not listed
    x[0, :, 1] = math.nan
    x[0, :, 2] = torch.finfo(torch.float32).min                        # ties of the lowest value: the lowest pages
    x[0, 2:7, 3] = -0.0
    x[0, 7:9, 3] = 0.0
    for sink, recent in ((1, 1), (0, 0)):
        want = ref.select_pages(x, cu, seq, 1, 5, 1, sink, recent)
        got = sp.select_pages(x.cuda(), cu.cuda(), _i32(seq).cuda(), kv_heads=1, topk=5, sink=sink, recent=recent)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("pages,total", [(8192, 2), (2000, 70), (300, 5000)])
def test_select_pages_of_long_sequences_and_many_tokens(sp, pages, total):
    gen = torch.Generator(device="cuda").manual_seed(pages)
    x = torch.randn((2, pages, total), device="cuda", generator=gen)
    seq = pages * PAGE
    got = sp.select_pages(x, _cu([total]).cuda(), _i32([seq]).cuda(), kv_heads=2, topk=20, causal=False)
    best = x.transpose(1, 2).clone()
    best[..., 0] = math.inf
    best[..., -1] = math.inf
    want = best.topk(20, -1).indices.sort(-1).values
    assert torch.equal(got.long(), want)


# ------------------------------------------------------------------ paged_attention
def _problem(seed, hkv, group, lens, seq, spare=3, q_scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    held = [-(-s // PAGE) for s in seq]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(seq), max(held + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    c = _cache(gen, pages, hkv, index=False)
    q = (q_scale * torch.randn((sum(lens), hkv * group, 128), generator=gen)).to(torch.bfloat16)
    return q, c, table, _i32(seq), _cu(lens)


def _random_ids(seed, hkv, lens, seq, topk, tile, total):
    rng = random.Random(seed)
    cu = _cu(lens)
    rows = total if tile == 1 else total // tile + len(lens)
    ids = torch.full((hkv, rows, topk), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        held = -(-seq[r] // PAGE)
        for i in range(-(-n // tile)):
            for h in range(hkv):
                some = sorted(rng.sample(range(held), min(held, rng.randint(0, topk))))
                ids[h, ref.list_row(int(cu[r]), r, i, tile), :len(some)] = _i32(some)
    return ids


def _check_attention(sp, q, c, table, seq, cu, ids=None, tile=1, causal=True, scale=None, max_q=None, gpu_q=None, floor=0.0, tiny=0.0):
    cache = _on_gpu(sp, c)
    total, hq = q.shape[:2]
    out = torch.full((total, hq, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((total, hq), 7.0, device="cuda")
    got, got_lse = sp.paged_attention(q.cuda() if gpu_q is None else gpu_q, cache, table.cuda(), seq.cuda(), cu.cuda(),
                                      None if ids is None else ids.cuda(), tile=tile, causal=causal, scale=scale,
                                      max_seqlen_q=max_q, out=out, lse=lse, return_lse=True)
    sp.device_status()
    assert got is out and got_lse is lse
    want, want_lse, spread, size = ref.paged_attention(q, c["k"], c["v"], c["k_scale"], c["v_scale"], table, seq, cu, ids, tile,
                                                       causal, scale)
    end = int(cu[-1])
    assert (out[end:] == 7).all() and (lse[end:] == 7).all()           # rows behind the last token stay
    out, lse, want, want_lse, spread, size = (x[:end] for x in (out.cpu().double(), lse.cpu().double(), want, want_lse, spread, size))
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(lse.isnan(), want_lse.isnan())
    assert torch.equal(lse == -math.inf, want_lse == -math.inf)
    ok, ok_l = ~want.isnan(), want_lse.isfinite()
    # Scores: 128 products are summed in 32 bits, each addition rounds by 2^-24 of the sum of magnitudes at most: 2^-17 of
    # sum |q k|; features of a query below 2^-22 of its largest lose up to 2^-23 of the largest: 128 of them 2^-16. So does the
    # natural-log LSE (2^-20 |lse| more for the logarithm and the exponentials).
    score = 2.0 ** -15 * size + 1e-6
    assert ((lse - want_lse).abs()[ok_l] <= (score + 2.0 ** -20 * want_lse.abs())[ok_l]).all()
    # Outputs: each probability carries exp(2 score error) and half a step of its 8-bit mantissa (2^-8), the output half a
    # step of bf16 (2^-8).
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * score[..., None]) * spread * 1.01 + 1e-30
    if floor:
        bound = bound + floor * spread.nan_to_num(0).amax(-1, keepdim=True) + tiny
    assert ((out - want).abs()[ok] <= bound[ok]).all(), ((out - want).abs() / bound)[ok].max()
    return out, lse


@pytest.mark.parametrize("hkv,group,lens,seq", [
    (1, 1, [1], [1]),
    (1, 1, [1], [128]),
    (2, 4, [1], [129]),
    (1, 16, [1, 1, 1], [700, 1, 255]),
    (3, 5, [1, 3, 0, 2], [127, 300, 9, 2]),
    (1, 3, [8, 8], [8, 1000]),
    (2, 8, [5, 1, 16], [5, 130, 400]),
    (1, 2, [200], [200]),                                              # a whole prompt
    (1, 64, [3], [260]),
    (1, 33, [2, 1], [140, 140]),
    (2, 1, [70, 3], [300, 3]),
    (1, 8, [1], [20000]),                                              # one long row
])
def test_attention_over_whole_sequences(sp, hkv, group, lens, seq):
    q, c, table, s, cu = _problem(11 + group, hkv, group, lens, seq)
    _check_attention(sp, q, c, table, s, cu, max_q=max(lens))
    if max(lens) > 1:
        _check_attention(sp, q, c, table, s, cu, max_q=1)              # a hint that is too small changes nothing
        _check_attention(sp, q, c, table, s, cu, causal=False)


@pytest.mark.parametrize("hkv,group,lens,seq,topk,tile", [
    (1, 16, [1, 1], [3000, 500], 7, 1),
    (3, 4, [2, 1, 8], [700, 1, 2000], 5, 1),
    (2, 8, [130, 5], [900, 400], 4, 16),
    (1, 16, [40, 3, 1], [1000, 3, 200], 3, 4),
    (1, 2, [300], [1500], 6, 128),
    (2, 5, [33, 9], [600, 600], 5, 8),
])
def test_attention_over_listed_pages(sp, hkv, group, lens, seq, topk, tile):
    q, c, table, s, cu = _problem(23 + group, hkv, group, lens, seq)
    ids = _random_ids(group, hkv, lens, seq, topk, tile, sum(lens))    # some lists are empty, some see nothing
    _check_attention(sp, q, c, table, s, cu, ids, tile, max_q=max(lens))
    _check_attention(sp, q, c, table, s, cu, ids, tile, causal=False)


def test_attention_with_odd_lists_tables_and_lengths(sp):
    q, c, table, s, cu = _problem(5, 1, 4, [2, 3, 1, 2], [400, 700, 300, 260])
    ids = torch.tensor([[0, 9, -3, 2], [2, 2, 1, 0], [5, 5, 5, 1 << 30], [-1, -1, -1, -1], [3, 1, 0, 4], [2, 1, -1, -1],
                        [0, 1, 2, 3], [1, -1, -1, -1]], dtype=torch.int32)[None]     # not pages, twice, none, any order
    table[1, 1], table[2, 1] = -5, c["k"].shape[0]                     # entries that name no page
    _check_attention(sp, q, c, table, s, cu, ids)
    s2 = _i32([1, 0, -4, 1 << 30])                                     # fewer keys than new tokens, none, beyond the table
    _check_attention(sp, q, c, table, s2, cu)
    _check_attention(sp, q, c, table, s2, cu, ids)


def test_attention_leaves_rows_behind_the_last_token(sp):
    q, c, table, s, cu = _problem(6, 2, 4, [3, 2], [200, 300])
    q = torch.cat([q, torch.full((6, 8, 128), math.nan, dtype=torch.bfloat16)])
    _check_attention(sp, q, c, table, s, cu)


def test_attention_from_strided_rows_and_another_scale(sp):
    q, c, table, s, cu = _problem(7, 2, 4, [3, 2], [200, 300])
    fused = torch.zeros((5, 14, 136), dtype=torch.bfloat16)
    fused[:, 3:11, :128] = q
    _check_attention(sp, q, c, table, s, cu, scale=0.3, gpu_q=fused.cuda()[:, 3:11, :128])
    _check_attention(sp, q, c, table, s, cu, scale=-0.1)
    _check_attention(sp, q, c, table, s, cu, scale=0.0)


def test_what_lies_behind_the_last_key_or_is_hidden_does_not_matter(sp):
    """NaN codes and scales behind the sequences and in pages that no list names; NaN rows that later tokens see only."""
    q, c, table, s, cu = _problem(8, 2, 4, [1, 4, 6], [200, 260, 130])
    want = _check_attention(sp, q, c, table, s, cu)
    nan = torch.tensor(0x7F, dtype=torch.uint8)
    for name in ("k", "v"):
        bits = c[name].view(torch.uint8)
        for r in range(3):
            n = int(s[r])
            if n % PAGE:
                bits[int(table[r, n // PAGE]), :, n % PAGE:] = nan
        used = set(table.flatten().tolist())
        for p in set(range(bits.shape[0])) - used:
            bits[p] = nan
            c[name + "_scale"][p] = math.nan
    got = _check_attention(sp, q, c, table, s, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for name in ("k", "v"):
        broken = {n: t.clone() for n, t in c.items()}
        bits = broken[name].view(torch.uint8)
        bits[int(table[1, 258 // PAGE]), :, 258 % PAGE, 5] = nan       # tokens 2 and 3 of request 1 see it
        bits[int(table[2, 1]), 1, 0, 9] = nan                          # tokens 4 and 5 of request 2, head 1
        out, _ = _check_attention(sp, q, broken, table, s, cu)
        assert torch.equal(out[:3], want[0][:3]) and not out[:3].isnan().any()


def test_attention_special_scores(sp):
    q, c, table, s, cu = _problem(9, 1, 2, [1, 2], [300, 150])
    c["k_scale"][int(table[0, 1])] = 1e4                               # one page takes everything
    c["v_scale"][int(table[0, 0])] = 1e30
    c["v_scale"][int(table[1, 0])] = 0.0
    q[1] = 0
    _check_attention(sp, q, c, table, s, cu)
    q[0, 0, 7] = math.nan                                              # a row of NaN stays by itself
    _check_attention(sp, q, c, table, s, cu)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 100.0, 1e30])
def test_attention_of_queries_of_any_size(sp, size):
    q, c, table, s, cu = _problem(10, 1, 4, [2], [300], q_scale=size)
    q[0, 1, ::2] *= 2.0 ** -9                                          # and of a row whose features differ widely
    q[0, 2, 5] *= 1000
    _check_attention(sp, q, c, table, s, cu, scale=0.05 / size)


def test_attention_in_a_graph_on_another_stream_and_twice_at_once(sp):
    q, c, table, s, cu = _problem(12, 2, 8, [1, 2, 1], [5000, 900, 20])
    cache = _on_gpu(sp, c)
    args = [t.cuda() for t in (table, s, cu)]
    gq = q.cuda()
    want = sp.paged_attention(gq, cache, *args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(sp.paged_attention(gq, cache, *args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    out = torch.empty_like(want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sp.paged_attention(gq, cache, *args, out=out)
        graphs.append(g)
    gq.copy_(gq.flip(0))
    args[1].copy_(_i32([900, 300, 2]).cuda())                          # other lengths: nothing of the plan is baked in
    want = sp.paged_attention(gq, cache, *args)
    for g in graphs:
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(sp):
    q, c, table, s, cu = _problem(13, 2, 4, [2], [300])
    cache = _on_gpu(sp, c)
    a = [t.cuda() for t in (q, table, s, cu)]
    call = lambda q=a[0], table=a[1], s=a[2], cu=a[3], **kw: sp.paged_attention(q, cache, table, s, cu, **kw)  # noqa: E731
    call()
    ids = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")
    for bad in (lambda: call(q=a[0].float()), lambda: call(q=a[0][:, :3]), lambda: call(q=a[0].cpu()),
                lambda: call(q=a[0][..., ::2]), lambda: call(s=a[2].long()), lambda: call(cu=a[3][:1]),
                lambda: call(table=a[1].t()), lambda: call(ids=ids[:1]), lambda: call(ids=ids, tile=3),
                lambda: call(ids=ids, tile=256), lambda: call(ids=ids.long()), lambda: call(out=a[0]),
                lambda: call(lse=torch.zeros(2, 8)), lambda: call(scale=math.nan), lambda: call(scale=math.inf),
                lambda: call(q=a[0].clone().requires_grad_()),
                lambda: call(q=torch.zeros((2, 130, 128), dtype=torch.bfloat16, device="cuda")),
                lambda: sp.PagedCache.from_tensors(cache.k, cache.v, cache.k_scale, cache.v_scale[:1]),
                lambda: sp.PagedCache(0, 1), lambda: sp.PagedCache(2, 0),
                lambda: sp.append_tokens(cache, a[0][:, :2], a[0][:, :3], a[3], torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: sp.append_tokens(cache, a[0][:, :2], a[0][:, :2], a[3], torch.zeros(2, dtype=torch.int32, device="cuda")),
                lambda: sp.append_tokens(cache, a[0][:, :2], a[0][:, :2], a[3], torch.zeros(3, dtype=torch.int64, device="cuda")),
                lambda: sp.select_pages(torch.zeros((2, 3, 2), device="cuda"), a[3], a[2], kv_heads=2, topk=1),
                lambda: sp.select_pages(torch.zeros((3, 3, 2), device="cuda"), a[3], a[2], kv_heads=2, topk=3),
                lambda: sp.select_pages(torch.zeros((2, 3, 2), device="cuda"), a[3], a[2], kv_heads=2, topk=3, tile=5),
                lambda: sp.select_pages(torch.zeros((2, 3, 2)), a[3], a[2], kv_heads=2, topk=3),
                lambda: sp.extend_pages(a[1], a[2], a[2].long(), a[2], a[2], total_q=1, total_pages=1),
                lambda: sp.extend_pages(a[1], a[2], a[2], a[2], a[2], total_q=-1, total_pages=1)):
        with pytest.raises(sp.SparseB200Error):
            bad()
    call()


# ------------------------------------------------------------------ the whole step
def test_steps_of_a_serving_loop(sp):
    """Prompts, then decode steps with a few tokens each: tables, cache, index, lists and attention as one, against the
    oracle of every stage on the stage's own inputs; the steps of the second half replay one graph."""
    gen = torch.Generator().manual_seed(77)
    hkv, group, batch, pages, width, topk = 2, 4, 3, 40, 12, 4
    cache = sp.PagedCache(pages, hkv, index=True)
    host = dict(k=torch.zeros((pages, hkv, PAGE, 128)), v=torch.zeros((pages, hkv, PAGE, 128)),
                k_scale=torch.ones((pages, hkv)), v_scale=torch.ones((pages, hkv)))
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(pages, generator=gen).to(torch.int32).cuda(), _i32([pages]).cuda()
    seq = torch.zeros(batch, dtype=torch.int32, device="cuda")
    for step, lens in enumerate(([300, 1, 700], [1, 1, 1], [3, 0, 2], [1, 130, 4])):
        total = sum(lens)
        b = sp.extend_pages(table, seq, _i32(lens).cuda(), free, count, total_q=total, total_pages=pages)
        assert int(b.status) == 0
        x = torch.randn((total, hkv * group + 2 * hkv, 128), generator=gen).to(torch.bfloat16)
        q, k, v = x[:, :hkv * group].contiguous(), x[:, hkv * group:-hkv], x[:, -hkv:]
        g = x.cuda()
        tile = 16 if step == 0 else 1
        out, ids = sp.paged_step(q.cuda(), g[:, hkv * group:-hkv], g[:, -hkv:], cache, table, b, topk=topk, tile=tile,
                                 max_seqlen_q=max(lens), max_seqlen_k=int(b.seq_lens.max()))
        for name, rows in (("k", k), ("v", v)):
            host[name], host[name + "_scale"] = ref.append_tokens(host[name], host[name + "_scale"], rows, b.cu_seqlens_q.cpu(),
                                                                  b.slots.cpu())
            assert torch.equal(getattr(cache, name).cpu().double(), host[name])
            assert torch.equal(getattr(cache, name + "_scale").cpu().double(), host[name + "_scale"])
        cu = b.cu_seqlens_q.cpu()
        qc, qs = sp.quantize_rows(q.cuda(), hkv)
        want_c, want_s = oracle.quantize_nvfp4(oracle.group_mean(q.transpose(0, 1)[None], hkv)[0].transpose(0, 1))
        assert torch.equal(qc.cpu(), want_c) and torch.equal(_bits(qs), want_s.view(torch.uint8))
        scores = sp.fp4_block_scores_varlen(qc, cache.k_index, qs, cache.k_index_scale, b.cu_seqlens_q, b.cu_seqlens_k,
                                            b.cu_page_offsets, max_seqlen_q=max(lens), max_seqlen_k=int(b.seq_lens.max()),
                                            kv_indices=b.kv_indices, causal=True, exact=False)
        assert torch.equal(ids.cpu(), ref.select_pages(scores.cpu(), cu, b.seq_lens.cpu(), hkv, topk, tile))
        want, _, spread, size = ref.paged_attention(q, host["k"], host["v"], host["k_scale"], host["v_scale"], table.cpu(),
                                                    b.seq_lens.cpu(), cu, ids.cpu(), tile)
        # as in _check_attention
        bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * (2.0 ** -15 * size[..., None] + 1e-6)) * spread * 1.01 + 1e-30
        assert ((out.cpu().double() - want).abs() <= bound).all()
        dense, none = sp.paged_step(q.cuda(), g[:, hkv * group:-hkv], g[:, -hkv:], cache, table, b, max_seqlen_q=max(lens),
                                    max_seqlen_k=int(b.seq_lens.max()))
        assert none is None and torch.equal(
            dense, sp.paged_attention(q.cuda(), cache, table, b.seq_lens, b.cu_seqlens_q, max_seqlen_q=max(lens)))
        seq, count = b.seq_lens, b.free_count


def test_a_step_in_a_graph(sp):
    """extend, append, score, select and attend captured once, replayed with other tokens and lengths."""
    gen = torch.Generator().manual_seed(78)
    hkv, group, batch, pages, width, topk, total = 1, 8, 2, 24, 8, 3, 4
    cache = [sp.PagedCache(pages, hkv) for _ in range(2)]
    for c in cache:
        c.k.view(torch.uint8).copy_(torch.randint(0, 0x70, c.k.shape, generator=gen).to(torch.uint8) if c is cache[0]
                                    else cache[0].k.view(torch.uint8))
        c.v.view(torch.uint8).copy_(cache[0].k.view(torch.uint8))
        c.k_index.copy_(cache[0].k.view(torch.uint8)[..., :64])
        c.k_index_scale.view(torch.uint8).fill_(0x38)
    table = [torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8) for _ in range(2)]
    free, count = torch.arange(16, 24, dtype=torch.int32, device="cuda"), _i32([8]).cuda()
    seq, new = _i32([300, 500]).cuda(), _i32([1, 3]).cuda()
    q = torch.randn((total, hkv * group, 128), generator=gen).to(torch.bfloat16).cuda()
    kv = torch.randn((2, total, hkv, 128), generator=gen).to(torch.bfloat16).cuda()

    def step(i):
        b = sp.extend_pages(table[i], seq, new, free, count, total_q=total, total_pages=pages)
        out, ids = sp.paged_step(q, kv[0], kv[1], cache[i], table[i], b, topk=topk, max_seqlen_q=4, max_seqlen_k=width * PAGE)
        return out, ids, b.slots, b.status
    step(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(0)
    for lens, added in (([300, 500], [1, 3]), ([639, 2], [2, 2]), ([0, 1020], [0, 4])):
        seq.copy_(_i32(lens))
        new.copy_(_i32(added))
        q.copy_(torch.randn(q.shape, generator=gen).to(torch.bfloat16))
        kv.copy_(torch.randn(kv.shape, generator=gen).to(torch.bfloat16))
        want = step(1)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(_bits(cache[0].k), _bits(cache[1].k)) and torch.equal(cache[0].k_scale, cache[1].k_scale)


# ------------------------------------------------------------------ items of many rows
_MANY_ROWS = [(1, 16, [20, 3], [700, 150]), (2, 40, [3, 1, 2], [390, 129, 300]), (1, 64, [5], [513])]


@pytest.mark.parametrize("hkv,group,lens,seq", _MANY_ROWS)
def test_attention_of_many_rows_special_scores(sp, hkv, group, lens, seq):
    q, c, table, s, cu = _problem(31 + group, hkv, group, lens, seq)
    # The weights of these items have 16 bits, 2^6 and more for the row's largest product W of probability and scale: one below
    # 2^-14 is off by 2^-25, half the smallest step, so by 2^-31 W. An output sums that over its keys, times codes of 448 at
    # most. W times the largest code of its key is among the row's spreads. A
    # probability below 2^-126 of the row's largest is 0 where parts are joined in 32 bits, whatever its value's scale.
    floor = max(seq) * 448 * 2.0 ** -31 / c["v"].float().abs().amax(-1).min().item()
    first, second = int(table[0, 0]), int(table[0, 1])
    for scales in ((1.0, 1e4, 1e30, 1.0), (1e4, 1.0, 1.0, 1e30), (1.0, 1.0, 1e-30, 1e30), (1.0, 1.0, 0.0, 1.0), (0.0, 1.0, 1.0, 0.0),
                   (30.0, 60.0, 2.0, 3.0), (1.0, 1.0, 1.0, 0.0)):
        c["k_scale"][first], c["k_scale"][second], c["v_scale"][first], c["v_scale"][second] = scales
        tiny = max(seq) * 448 * 2.0 ** -126 * max(scales[2:])
        _check_attention(sp, q, c, table, s, cu, max_q=max(lens), floor=floor, tiny=tiny)
        _check_attention(sp, q, c, table, s, cu, max_q=max(lens), causal=False, floor=floor, tiny=tiny)
    c["v_scale"][:] = 0.0
    _check_attention(sp, q, c, table, s, cu, max_q=max(lens))
    c["v_scale"][:] = 1.0
    q[0, 1] = 0
    q[-1, group - 1, 7] = math.nan                                     # a row of NaN stays by itself
    _check_attention(sp, q, c, table, s, cu, max_q=max(lens), scale=-0.2, floor=floor)


@pytest.mark.parametrize("hkv,group,lens,seq", _MANY_ROWS)
def test_attention_of_many_rows_hidden_nan(sp, hkv, group, lens, seq):
    """NaN codes in keys and values that some of an item's rows see, and behind the sequence."""
    q, c, table, s, cu = _problem(37 + group, hkv, group, lens, seq)
    want = _check_attention(sp, q, c, table, s, cu, max_q=max(lens))
    nan = torch.tensor(0x7F, dtype=torch.uint8)
    for name in ("k", "v"):
        bits = c[name].view(torch.uint8)
        for r, n in enumerate(seq):
            if n % PAGE:
                bits[int(table[r, n // PAGE]), :, n % PAGE:] = nan
    got = _check_attention(sp, q, c, table, s, cu, max_q=max(lens))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    last = seq[0] - 1                                                  # only the last token of request 0 sees it
    for name in ("k", "v"):
        broken = {n: t.clone() for n, t in c.items()}
        broken[name].view(torch.uint8)[int(table[0, last // PAGE]), hkv - 1, last % PAGE, 77] = nan
        out, _ = _check_attention(sp, q, broken, table, s, cu, max_q=max(lens))
        assert out[lens[0] - 1].isnan().any() and torch.equal(out[:lens[0] - 1], want[0][:lens[0] - 1])


def test_attention_of_many_short_items(sp):
    """Items of a page each: the roles of a CTA are items apart. The same bits every time, whatever the hint."""
    lens, seq = [9, 1, 2, 2, 0, 35, 35, 0, 19, 0], [9, 1327, 2, 122, 101, 1401, 287, 0, 19, 1151]
    q, c, table, s, cu = _problem(41, 2, 40, lens, seq)
    for max_q in (1, None):
        _check_attention(sp, q, c, table, s, cu, max_q=max_q)
        cache, args = _on_gpu(sp, c), [t.cuda() for t in (table, s, cu)]
        first = sp.paged_attention(q.cuda(), cache, *args, max_seqlen_q=max_q)
        gq = q.cuda()
        for _ in range(200):
            assert torch.equal(sp.paged_attention(gq, cache, *args, max_seqlen_q=max_q), first)


def test_attention_of_many_rows_in_a_graph_on_another_stream_and_twice_at_once(sp):
    q, c, table, s, cu = _problem(43, 1, 8, [70, 16, 1], [5000, 900, 20])
    ids = _random_ids(3, 1, [70, 16, 1], [5000, 900, 20], 6, 16, 87).cuda()
    cache, args, gq = _on_gpu(sp, c), [t.cuda() for t in (table, s, cu)], q.cuda()
    for kw in (dict(), dict(ids=ids, tile=16)):
        want = sp.paged_attention(gq, cache, *args, **kw)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for _ in range(10):
            for st in streams:
                with torch.cuda.stream(st):
                    got.append(sp.paged_attention(gq, cache, *args, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
        out, graphs = torch.empty_like(want), []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                sp.paged_attention(gq, cache, *args, out=out, **kw)
            graphs.append(g)
        for g in graphs + graphs:
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("hkv,group,lens,seq", [(2, 4, [4], [130]), (1, 40, [4], [130])])
def test_attention_scale_of_a_page_that_some_tokens_do_not_see(sp, hkv, group, lens, seq):
    q, c, table, s, cu = _problem(47, hkv, group, lens, seq)
    want = _check_attention(sp, q, c, table, s, cu)
    for name in ("k_scale", "v_scale"):
        for bad in (math.nan, math.inf):
            broken = {n: t.clone() for n, t in c.items()}
            broken[name][int(table[0, 1])] = bad                       # tokens 2 and 3 see the second page
            cache = _on_gpu(sp, broken)
            for max_q in (1, 4):
                out, lse = sp.paged_attention(q.cuda(), cache, table.cuda(), s.cuda(), cu.cuda(), max_seqlen_q=max_q,
                                              return_lse=True)
                assert torch.equal(out[:2].cpu().double(), want[0][:2]) and torch.equal(lse[:2].cpu().double(), want[1][:2])


@pytest.mark.parametrize("group,tokens", [(4, 1), (16, 8)])
def test_attention_of_shares_of_many_pages(sp, group, tokens):
    """More than 32 pages of an item in a share. Requests are alike, over the same pages."""
    hkv, batch, keys = 2, 64, 64 * PAGE - 5
    q, c, table, s, cu = _problem(53, hkv, group, [tokens], [keys])
    want, want_lse, spread, size = ref.paged_attention(q, c["k"], c["v"], c["k_scale"], c["v_scale"], table, s, cu)
    lens = [tokens] * (batch * 5)
    out, lse = sp.paged_attention(q.repeat(len(lens), 1, 1).cuda(), _on_gpu(sp, c), table.repeat(len(lens), 1).cuda(),
                                  s.repeat(len(lens)).cuda(), _cu(lens).cuda(), max_seqlen_q=tokens, return_lse=True)
    sp.device_status()
    out = out.view(len(lens), tokens, hkv * group, 128).cpu().double()
    lse = lse.view(len(lens), tokens, hkv * group).cpu().double()
    # as in _check_attention
    score = 2.0 ** -15 * size + 1e-6
    assert ((lse - want_lse).abs() <= score + 2.0 ** -20 * want_lse.abs()).all()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * score[..., None]) * spread * 1.01 + 1e-30
    assert ((out - want).abs() <= bound).all()


def test_attention_of_many_rows_strided_and_padded(sp):
    q, c, table, s, cu = _problem(59, 2, 4, [30, 12], [200, 300])
    q = torch.cat([q, torch.full((6, 8, 128), math.nan, dtype=torch.bfloat16)])
    _check_attention(sp, q, c, table, s, cu)                           # rows behind the last token stay
    fused = torch.full((48, 14, 136), math.nan, dtype=torch.bfloat16)
    fused[:, 3:11, :128] = q
    _check_attention(sp, q, c, table, s, cu, scale=0.3, gpu_q=fused.cuda()[:, 3:11, :128])
    _check_attention(sp, q, c, table, s, cu, scale=0.0)


@pytest.mark.parametrize("hkv,group,lens,seq", [(1, 4, [2], [500]), (1, 16, [20], [700])])
def test_attention_of_huge_scores(sp, hkv, group, lens, seq):
    """Scores whose differences are beyond 32 bits: the rows stay finite, within the values that they see."""
    q, c, table, s, cu = _problem(61, hkv, group, lens, seq)
    for scale in (1e4, 1e6, 1e8, 1e12, 1e30):
        cache = _on_gpu(sp, c)
        out, lse = sp.paged_attention(q.cuda(), cache, table.cuda(), s.cuda(), cu.cuda(), scale=scale, return_lse=True)
        assert out.isfinite().all() and lse.isfinite().all()
        most = (c["v"].float().abs() * c["v_scale"][..., None, None].float()).max().item()
        assert out.abs().max() <= 1.01 * most
        _check_attention(sp, q, c, table, s, cu, scale=scale)
