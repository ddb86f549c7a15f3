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
