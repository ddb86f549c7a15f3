"""The operators of the paged serving path, as cases that can be timed and compared.

  extend     page tables, slot map and cumulative lengths of a step from the requests' lengths
  append     keys and values of the new tokens into 8-bit pages with a scale per page and head, and their NVFP4 index vectors
  select     page scores of the new tokens -> lists of pages
  attention  new tokens over the 8-bit pages of their requests, all of them or the listed ones

A page holds 128 tokens and a head has 128 features. Request lengths are part of a case (drawn from its `lengths`);
everything else that is random is drawn on the GPU from the seed. With `own` the framework's entry points run, without
it their plain form in elementary torch operations."""
import math
import random

import torch

own = False

PAGE, D = 128, 128
E4M3_MAX, LOWEST_EXPONENT = 448.0, -100


def listed():
    return [
        # a decode step of 48 requests: one new token each, a page now and then; latency is all there is
        dict(name="extend_decode", op="extend", requests=48, q_lo=1, q_hi=1, k_lo=1, k_hi=32768, lengths=3),
        # a large mixed batch, up to 128 new tokens each
        dict(name="extend_mixed", op="extend", requests=768, q_lo=0, q_hi=128, k_lo=0, k_hi=32768, lengths=5),
        # a decode batch with a few (speculated) tokens for each request
        dict(name="append_decode", op="append", requests=64, hkv=4, q_lo=1, q_hi=8, k_lo=0, k_hi=4096, index=True, lengths=7),
        # ragged prompts, some of them continued within a page
        dict(name="append_prefill", op="append", requests=8, hkv=4, q_lo=512, q_hi=4096, k_lo=0, k_hi=2048, index=True,
             lengths=7),
        # lists of a decode batch of long requests: 16 index heads of one key head, a few new tokens each
        dict(name="select_decode", op="select", requests=64, hkv=1, group=16, q_lo=1, q_hi=8, k_lo=8192, k_hi=32768,
             tile=1, topk=64, lengths=7),
        # lists of every token of ragged prompts
        dict(name="select_prefill", op="select", requests=8, hkv=2, group=1, q_lo=512, q_hi=4096, k_lo=4096, k_hi=16384,
             tile=1, topk=16, lengths=7),
        # the smallest attention: one new token of one short request
        dict(name="attention_one", op="attention", requests=1, hkv=2, group=4, q_lo=1, q_hi=1, k_lo=700, k_hi=700, tile=1,
             topk=0, lengths=1),
        # speculated tokens of short and middling requests, whole sequences
        dict(name="attention_speculative", op="attention", requests=32, hkv=8, group=4, q_lo=1, q_hi=8, k_lo=1, k_hi=8192,
             tile=1, topk=0, lengths=9),
        # a decode batch of long requests over 64 selected pages each
        dict(name="attention_sparse_decode", op="attention", requests=64, hkv=4, group=16, q_lo=1, q_hi=1, k_lo=8192,
             k_hi=32768, tile=1, topk=64, lengths=7),
        # the same batch over whole sequences
        dict(name="attention_dense_decode", op="attention", requests=64, hkv=4, group=16, q_lo=1, q_hi=1, k_lo=8192,
             k_hi=32768, tile=1, topk=0, lengths=7),
        # one request of 1 Mi tokens: a single long row to be split over the GPU
        dict(name="attention_long", op="attention", requests=1, hkv=1, group=8, q_lo=1, q_hi=1, k_lo=1048576, k_hi=1048576,
             tile=1, topk=0, lengths=1),
        # chunks of prompts over longer contexts, every 16 tokens share a list
        dict(name="attention_prefill_tiles", op="attention", requests=4, hkv=1, group=16, q_lo=512, q_hi=1024, k_lo=4096,
             k_hi=16384, tile=16, topk=16, lengths=7),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    while True:
        op = rng.choice(["extend", "append", "select", "attention", "attention", "attention"])
        q_hi = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 4096)])
        k_hi = _log(rng, max(64, q_hi), 65536)
        case = dict(op=op, requests=_log(rng, 1, 768 if op == "extend" else 96), q_lo=max(1, q_hi // 8), q_hi=q_hi,
                    k_lo=max(1, k_hi // rng.choice([2, 4, 64])), k_hi=k_hi, lengths=rng.randrange(1 << 20))
        if op != "extend":
            case["hkv"] = rng.choice([1, 1, 2, 3, 4, 8])
        if op == "append":
            case["index"] = rng.random() < 0.7
        if op in ("select", "attention"):
            case.update(group=rng.choice([1, 2, 3, 4, 5, 8, 16]), tile=1, topk=_log(rng, 3, 64))
            if q_hi > 8:
                case["tile"] = rng.choice([1, 4, 16, 64])
            if op == "attention" and rng.random() < 0.5:
                case.update(tile=1, topk=0)
            if op == "select":
                # sequences that have more pages than a list takes
                case["k_lo"] = max(case["k_lo"], (case["topk"] + 2) * PAGE)
                case["k_hi"] = max(case["k_hi"], case["k_lo"])
        w = work(case)
        flops, bytes_ = {"extend": (1, 1e8), "append": (1, 2.5e8), "select": (1, 2e8), "attention": (6e11, 1.4e9)}[op]
        if w["flops"] <= flops and w["bytes"] <= bytes_ and _plain_bytes(case) <= 2e10:
            return case


def _lengths(case):
    """New tokens and cached tokens (without the new ones where the step appends, else with them) of every request."""
    r = random.Random(case["lengths"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["requests"])]
    k = [r.randint(case["k_lo"], case["k_hi"]) for _ in q]
    if case["op"] in ("select", "attention"):
        k = [max(n, m) for n, m in zip(q, k)]
    return q, k


def _plain_bytes(case):
    """What the plain form of a case holds at its largest, about."""
    q, k = _lengths(case)
    if case["op"] == "attention":
        if case["topk"]:
            rows = sum(-(-n // case["tile"]) for n in q)
            return rows * case["hkv"] * case["topk"] * PAGE * (3 * 4 * D + 12 * case["tile"] * case["group"])
        return len(q) * max(k) * case["hkv"] * (3 * 4 * D + 12 * max(q) * case["group"])
    if case["op"] == "select":
        return 30 * sum(q) * -(-max(k) // PAGE) * case["hkv"] * case["group"]
    return 0


def _pages(n):
    return -(-n // PAGE)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cumulated(x):
    return torch.tensor([0] + list(x), device="cuda").cumsum(0).to(torch.int32)


def _codes(shape, gen):
    """e4m3 codes of N(0, 1) values at a scale that brings their largest near 448, as the cache holds them."""
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat, step = out.view(-1), 1 << 28
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.empty(n, device="cuda").normal_(generator=gen).mul_(100).clamp_(-E4M3_MAX, E4M3_MAX).to(out.dtype)
    return out


def _scales(shape, gen):
    """Powers of two about 2^-7: the values behind the codes are about 1."""
    return torch.exp2(torch.randint(-8, -5, shape, device="cuda", generator=gen).float())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, (q_lens, k_lens) = case["op"], _lengths(case)
    n, s = len(q_lens), dict(op=case["op"], case=case)
    total = sum(q_lens)
    if op == "extend":
        width = _pages(case["k_hi"] + case["q_hi"]) + 1
        before, after = [_pages(k) for k in k_lens], [_pages(k + m) for k, m in zip(k_lens, q_lens)]
        order = torch.randperm(sum(after) + 64, device="cuda", generator=gen).to(torch.int32)    # 64 pages stay free
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        at = torch.arange(width, device="cuda")[None] < torch.tensor(before, device="cuda")[:, None]
        table[at] = order[:sum(before)]
        s.update(table=table, seq=_int32(k_lens), new=_int32(q_lens), free=order[sum(before):].contiguous(),
                 count=_int32([sum(after) + 64 - sum(before)]), total_q=total, total_pages=sum(after))
        return s
    if op == "select":
        tiles = _pages(max(k_lens))
        s.update(cu_q=_cumulated(q_lens), seq=_int32(k_lens))
        s["scores"] = torch.empty((case["hkv"] * case["group"], tiles, total), device="cuda").normal_(generator=gen).mul_(8)
        last = torch.tensor([k - q for q, k in zip(q_lens, k_lens)], device="cuda").repeat_interleave(
            torch.tensor(q_lens, device="cuda")) + torch.cat([torch.arange(m, device="cuda") for m in q_lens])
        s["scores"].masked_fill_(torch.arange(tiles, device="cuda")[:, None] * PAGE > last[None], -math.inf)
        return s
    held = [_pages(k + (m if op == "append" else 0)) for k, m in zip(k_lens, q_lens)]
    pages, hkv = sum(held), case["hkv"]
    table = torch.full((n, max(held)), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(max(held), device="cuda")[None] < torch.tensor(held, device="cuda")[:, None]] = \
        torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    for name in ("k", "v"):
        s[name] = _codes((pages, hkv, PAGE, D), gen)
        s[name + "_scale"] = _scales((pages, hkv), gen)
    s["cu_q"] = _cumulated(q_lens)
    if op == "append":
        x = torch.empty((2, total, hkv, D), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
        s["new_k"], s["new_v"] = x[0], x[1]
        position = torch.tensor(k_lens, device="cuda").repeat_interleave(torch.tensor(q_lens, device="cuda")) + torch.cat(
            [torch.arange(m, device="cuda") for m in q_lens])
        request = torch.arange(n, device="cuda").repeat_interleave(torch.tensor(q_lens, device="cuda"))
        s["slots"] = table[request, position // PAGE].long() * PAGE + position % PAGE
        s["k_index"] = s["k_index_scale"] = None
        if case["index"]:
            s["k_index"] = torch.randint(256, (pages, hkv, PAGE, D // 2), dtype=torch.uint8, device="cuda", generator=gen)
            s["k_index_scale"] = torch.ones((pages, hkv, PAGE, D // 16), device="cuda").to(torch.float8_e4m3fn)
    else:
        s.update(table=table, seq=_int32(k_lens), max_q=max(q_lens))
        s["q"] = torch.empty((total, hkv * case["group"], D), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
        s["ids"] = _lists(case, q_lens, k_lens, gen) if case["topk"] else None
    if own:
        import sparse_attention_b200_b200 as sp
        s["cache"] = sp.PagedCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"], s.get("k_index"),
                                                s.get("k_index_scale"))
    return s


def _list_rows(case, q_lens):
    """Row of every tile's list, and the request and the first token of the tile within it."""
    tile, rows, at = case["tile"], [], 0
    for r, n in enumerate(q_lens):
        first = at if tile == 1 else at // tile + r
        rows += [(first + i, r, i * tile) for i in range(-(-n // tile))]
        at += n
    return rows, (at if tile == 1 else at // tile + len(q_lens))


def _lists(case, q_lens, k_lens, gen):
    """Distinct pages that the last token of a tile sees, ascending, the first and the last among them; -1 behind."""
    rows, count = _list_rows(case, q_lens)
    tile, topk, most = case["tile"], case["topk"], _pages(max(k_lens))
    seen = torch.tensor([_pages(k_lens[r] - q_lens[r] + min(i + tile, q_lens[r])) for _, r, i in rows], device="cuda")
    at = torch.tensor([row for row, _, _ in rows], device="cuda")
    ids = torch.full((case["hkv"], count, topk), -1, dtype=torch.int32, device="cuda")
    page = torch.arange(most, device="cuda")
    for h in range(case["hkv"]):
        x = torch.rand((len(rows), most), device="cuda", generator=gen)
        x.masked_fill_((page == 0) | (page == seen[:, None] - 1), 2.0).masked_fill_(page >= seen[:, None], -1.0)
        value, index = x.topk(min(topk, most), 1)
        index = index.masked_fill(value < 0, most).sort(1).values
        ids[h, at, :index.shape[1]] = index.masked_fill(index == most, -1).int()
    return ids


def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


# ------------------------------------------------------------------ the framework's entry points
def _own_extend(s):
    import sparse_attention_b200_b200 as sp
    b = sp.extend_pages(s["table"], s["seq"], s["new"], s["free"], s["count"], total_q=s["total_q"],
                        total_pages=s["total_pages"])
    return (s["table"], b.seq_lens, b.cu_seqlens_q, b.cu_seqlens_k, b.cu_page_offsets, b.kv_indices, b.slots, b.free_count,
            b.status)


def _own_append(s):
    import sparse_attention_b200_b200 as sp
    sp.append_tokens(s["cache"], s["new_k"], s["new_v"], s["cu_q"], s["slots"])
    return s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_index"], s["k_index_scale"]


def _own_select(s):
    import sparse_attention_b200_b200 as sp
    c = s["case"]
    return sp.select_pages(s["scores"], s["cu_q"], s["seq"], kv_heads=c["hkv"], topk=c["topk"], tile=c["tile"])


def _own_attention(s):
    import sparse_attention_b200_b200 as sp
    return sp.paged_attention(s["q"], s["cache"], s["table"], s["seq"], s["cu_q"], ids=s["ids"], tile=s["case"]["tile"],
                              max_seqlen_q=s["max_q"], return_lse=True)


# ------------------------------------------------------------------ the plain forms
def _zero_cumsum(x):
    return torch.nn.functional.pad(x.cumsum(0), (1, 0)).int()


def _plain_extend(s):
    old, new, table, free = s["seq"].clamp(min=0), s["new"].clamp(min=0), s["table"], s["free"]
    n, width = table.shape
    total_q, total_pages = s["total_q"], s["total_pages"]
    before, after = (old + PAGE - 1) // PAGE, (old + new + PAGE - 1) // PAGE
    wide = after > width
    need = torch.where(wide, 0, after - before)
    upto = need.cumsum(0).int()
    short = (need > 0) & (upto > s["count"])
    granted = ~(wide | short)
    k = old + torch.where(granted, new, 0)
    pages = (k + PAGE - 1) // PAGE
    column = torch.arange(width, device="cuda")[None]
    fresh = (column >= before[:, None]) & (column < after[:, None]) & granted[:, None]
    at = s["count"] - 1 - (upto - need)[:, None] - (column - before[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    cu_q, cu_k, cu_pages = _zero_cumsum(new), _zero_cumsum(k), _zero_cumsum(pages)
    t = torch.arange(total_q, device="cuda")
    r = torch.searchsorted(cu_q[1:].contiguous(), t.int(), right=True)
    live, r = r < n, r.clamp(max=n - 1)
    p = old[r] + t.int() - cu_q[r]
    page = table[r, (p // PAGE).clamp(max=width - 1)]
    slots = torch.where(live & granted[r] & (page >= 0), page.long() * PAGE + p % PAGE, -1)
    j = torch.arange(total_pages, device="cuda", dtype=torch.int32)
    r = torch.searchsorted(cu_pages[1:].contiguous(), j, right=True)
    live, r = r < n, r.clamp(max=n - 1)
    kv_indices = torch.where(live, table[r, (j - cu_pages[r]).clamp(max=width - 1)], -1)
    count = s["count"] - torch.where(granted, need, 0).sum().int()
    status = (short.any().int() + 2 * wide.any().int() + 4 * (cu_q[-1:] > total_q).int() + 8 * (cu_pages[-1:] > total_pages).int())
    return table, k, cu_q, cu_k, cu_pages, kv_indices, slots, count, status


def _e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _plain_store(x, cache, scale, first_page, first_offset, page, offset):
    """The rows x [T, hkv, D] (32 bits) at (page, offset) of the cache; the scales of their pages with them."""
    pages, hkv = scale.shape
    top = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(top)
    exponent = torch.where(top > 0, exponent - torch.where(mantissa <= 0.875, 9, 8), LOWEST_EXPONENT)
    need = torch.exp2(exponent.clamp(min=LOWEST_EXPONENT).float())
    touched = torch.zeros(pages, dtype=torch.bool, device="cuda")
    touched[page] = True
    prior = torch.zeros_like(touched)
    prior[first_page] = first_offset > 0
    grown = torch.where(prior[:, None], torch.maximum(need, scale), need)
    grown = torch.where(touched[:, None], grown, scale)
    # rows before the new ones keep their values at the new scale
    held = cache[first_page].float() * (scale / grown)[first_page][..., None, None]
    keep = torch.arange(PAGE, device="cuda")[None, None, :, None] < first_offset[:, None, None, None]
    bits = cache.view(torch.uint8)
    bits[first_page] = torch.where(keep, _e4m3(held).view(torch.uint8), bits[first_page])
    scale.copy_(grown)
    bits[page, :, offset] = _e4m3(x / grown[page][..., None]).view(torch.uint8)


def _plain_nvfp4(x):
    """x [..., D] (32 bits) -> packed e2m1 codes and one e4m3 scale per 16 features."""
    groups = x.unflatten(-1, (-1, 16))
    scale = (groups.abs().amax(-1) / 6.0).clamp(max=E4M3_MAX).to(torch.float8_e4m3fn)
    step = scale.float()[..., None]
    ratio = torch.where(step > 0, groups / torch.where(step > 0, step, 1.0), 0.0).flatten(-2)
    a = ratio.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() +
            (a >= 3.5).byte() + (a > 5.0).byte())
    code = code + 8 * ((ratio < 0) & (code > 0)).byte()
    return code[..., 0::2] + 16 * code[..., 1::2], scale


def _plain_append(s):
    page, offset = s["slots"] // PAGE, s["slots"] % PAGE
    first = s["slots"][s["cu_q"][:-1].long()]
    for name in ("k", "v"):
        _plain_store(s["new_" + name].float(), s[name], s[name + "_scale"], first // PAGE, first % PAGE, page, offset)
    if s["k_index"] is not None:
        codes, scales = _plain_nvfp4(s["new_k"].float())
        s["k_index"][page, :, offset] = codes
        s["k_index_scale"].view(torch.uint8)[page, :, offset] = scales.view(torch.uint8)
    return s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_index"], s["k_index_scale"]


def _tiles(cu_q, tile, total):
    """For every token: the row of its tile's list; and how many rows there are."""
    n = cu_q.numel() - 1
    t = torch.arange(total, device="cuda", dtype=torch.int32)
    r = torch.searchsorted(cu_q[1:].contiguous(), t, right=True)
    if tile == 1:
        return r, t.long(), total
    return r, cu_q[r].long() // tile + r + (t - cu_q[r]).long() // tile, total // tile + n


def _plain_select(s):
    c, scores, cu_q, seq = s["case"], s["scores"], s["cu_q"], s["seq"]
    hkv, topk, tile = c["hkv"], c["topk"], c["tile"]
    pages, total = scores.shape[1:]
    x = scores.view(hkv, -1, pages, total).nan_to_num(-math.inf, math.inf, -math.inf).amax(1)
    request, row, rows = _tiles(cu_q, tile, total)
    last = (seq[request] - cu_q[1:][request]).long() + torch.arange(total, device="cuda")
    best = torch.full((hkv, pages, rows), -math.inf, device="cuda")
    best.scatter_reduce_(2, row[None, None].expand(hkv, pages, total), x, "amax")
    seen = torch.zeros(rows, dtype=torch.long, device="cuda").scatter_reduce_(0, row, last // PAGE + 1, "amax")
    page = torch.arange(pages, device="cuda")[:, None]
    always = ((page < 1) | (page >= seen - 1)) & (page < seen)
    best.masked_fill_(always, math.inf).masked_fill_(page >= seen, -math.inf)
    value, index = best.transpose(1, 2).sort(dim=2, descending=True, stable=True)
    value, index = value[..., :topk], index[..., :topk]
    index = index.masked_fill(value == -math.inf, pages).sort(2).values
    ids = torch.full((hkv, rows, topk), -1, dtype=torch.int32, device="cuda")
    ids[..., :index.shape[2]] = index.masked_fill(index == pages, -1)
    return ids


def _plain_attention(s):
    c, q, table, seq, cu_q, ids = s["case"], s["q"], s["table"], s["seq"], s["cu_q"], s["ids"]
    total, hq = q.shape[:2]
    hkv, n = c["hkv"], seq.numel()
    tile = c["tile"] if ids is not None else s["max_q"]
    # one row for each tile of a request: its tokens, padded, against the pages that it reads
    request, row, rows = _tiles(cu_q, tile, total)
    if ids is None and tile > 1:
        row, rows = request, n
    within = (torch.arange(total, device="cuda") - cu_q[request]) % tile if tile > 1 else torch.zeros_like(row)
    place = row * tile + within
    rows_q = torch.zeros((rows * tile, hq, D), device="cuda").index_copy_(0, place, q.float())
    rows_q = rows_q.view(rows, tile, hkv, -1, D).transpose(1, 2).flatten(2, 3)
    last = torch.full((rows * tile,), -1, dtype=torch.long, device="cuda").index_copy_(
        0, place, (seq[request] - cu_q[1:][request]).long() + torch.arange(total, device="cuda")).view(rows, 1, tile, 1, 1)
    owner = torch.zeros(rows, dtype=torch.long, device="cuda").index_copy_(0, row, request)
    if ids is None:
        pages = torch.arange(table.shape[1], device="cuda").expand(rows, hkv, -1)
    else:
        pages = ids.transpose(0, 1).long()
    held = table[owner[:, None, None], pages.clamp(min=0)].long().clamp(min=0)
    head = torch.arange(hkv, device="cuda")[None, :, None]
    key = (pages[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(2).masked_fill(
        (pages < 0).repeat_interleave(PAGE, 2), 1 << 40)

    def values(codes, scale):
        x = codes.view(torch.uint8)[held, head].view(torch.float8_e4m3fn).float()
        return x.mul_(scale[held, head][..., None, None]).flatten(2, 3)
    x = rows_q @ values(s["k"], s["k_scale"]).transpose(2, 3)
    x = x.mul_(1 / math.sqrt(D)).view(rows, hkv, tile, -1, key.shape[2])
    x.masked_fill_(key[:, :, None, None] > last, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(top).exp_()
    sums = x.sum(-1, keepdim=True)
    out = (x.flatten(2, 3) @ values(s["v"], s["v_scale"])).view(rows, hkv, tile, -1, D) / sums
    lse = (top + sums.log()).squeeze(-1)
    out = out.transpose(1, 2).reshape(rows * tile, hq, D)[place]
    return out.to(torch.bfloat16), lse.transpose(1, 2).reshape(rows * tile, hq)[place]


_run_own = dict(extend=_own_extend, append=_own_append, select=_own_select, attention=_own_attention)
_run_plain = dict(extend=_plain_extend, append=_plain_append, select=_plain_select, attention=_plain_attention)


def work(case):
    op, (q_lens, k_lens) = case["op"], _lengths(case)
    total = sum(q_lens)
    if op == "extend":
        pages = sum(_pages(k + m) for k, m in zip(k_lens, q_lens))
        fresh = pages - sum(_pages(k) for k in k_lens)
        return {"bytes": 8 * pages + 4 * fresh + 8 * total + 24 * len(q_lens), "flops": 0.0}
    hkv = case["hkv"]
    if op == "append":
        return {"bytes": total * hkv * (2 * (2 * D + D) + (72 if case["index"] else 0)) + 8 * total, "flops": 0.0}
    rows = _list_rows(case, q_lens)[0]
    if op == "select":
        # scores of the pages that a token sees
        seen = sum((n * m - n * (n - 1) // 2) / PAGE + n / 2 for n, m in zip(q_lens, k_lens))
        return {"bytes": 4 * hkv * (case["group"] * seen + len(rows) * case["topk"]), "flops": 0.0}
    tile, topk, group = case["tile"], case["topk"], case["group"]
    page = 2 * (PAGE * D + 4)
    if topk:
        # distinct pages of a request that its lists name, for lists drawn at random, and the keys of a list
        read = pairs = 0
        for _, r, i in rows:
            tokens = min(tile, q_lens[r] - i)
            pairs += tokens * min(topk * PAGE, k_lens[r] - q_lens[r] + i + (tokens + 1) / 2)
        for n, m in zip(q_lens, k_lens):
            lists = -(-n // tile)
            read += _pages(m) * (1 - (1 - min(1.0, topk / _pages(m))) ** lists)
    else:
        read = sum(_pages(m) for m in k_lens)
        pairs = sum(n * m - n * (n - 1) // 2 for n, m in zip(q_lens, k_lens))
    hq = hkv * group
    ids = 4 * hkv * len(rows) * topk
    return {"bytes": read * hkv * page + total * hq * (4 * D + 4) + ids, "flops": 4.0 * D * hq * pairs}


# ------------------------------------------------------------------ 64 bits
def _nearest_e4m3(x):
    """The e4m3 value nearest to x (ties to the even code), saturated; 64 bits."""
    exponent = torch.frexp(x)[1].sub(1).clamp(min=-6)
    step = torch.exp2((exponent - 3).double())
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(s, case):
    q_lens, k_lens = _lengths(case)
    answer = []
    for name in ("k", "v"):
        x, codes, scale = s["new_" + name].double(), s[name].double(), s[name + "_scale"].double()
        at = 0
        for n, m in zip(q_lens, k_lens):
            done = 0
            while done < n:
                page, o = divmod(int(s["slots"][at + done]), PAGE)
                count = min(PAGE - o, n - done)
                rows = x[at + done:at + done + count].transpose(0, 1)
                top = rows.abs().amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=LOWEST_EXPONENT))
                if o:
                    need = torch.maximum(need, scale[page])
                    codes[page, :, :o] = _nearest_e4m3(codes[page, :, :o] * (scale[page] / need)[:, None, None])
                scale[page] = need
                codes[page, :, o:o + count] = _nearest_e4m3(rows / need[:, None, None])
                done += count
            at += n
        answer.append((codes, scale))
    (k, ks), (v, vs) = answer
    return k, v, ks, vs, None, None


def _exact_attention(s, case):
    q_lens, k_lens = _lengths(case)
    hkv, group, tile = case["hkv"], case["group"], case["tile"]
    out = torch.empty((sum(q_lens), hkv * group, D), dtype=torch.float64, device="cuda")
    lse = torch.empty((sum(q_lens), hkv * group), dtype=torch.float64, device="cuda")
    rows = _list_rows(case, q_lens)[0] if case["topk"] else [(0, r, 0) for r in range(len(q_lens))]
    lists = s["ids"].tolist() if case["topk"] else None
    start = [sum(q_lens[:r]) for r in range(len(q_lens))]
    table = s["table"].long()
    for row, r, first in rows:
        count = min(tile, q_lens[r] - first) if lists else q_lens[r]
        for h in range(hkv):
            pages = [j for j in lists[h][row] if j >= 0] if lists else list(range(_pages(k_lens[r])))
            logical = torch.tensor(pages, device="cuda")
            held = table[r, logical]
            k, v = (s[a][held, h].double() * s[a + "_scale"][held, h].double()[:, None, None] for a in ("k", "v"))
            key = (logical[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()
            at, heads = slice(start[r] + first, start[r] + first + count), slice(h * group, (h + 1) * group)
            q = s["q"][at, heads].double()
            last = k_lens[r] - q_lens[r] + first + torch.arange(count, device="cuda")
            x = torch.einsum("tgd,kd->tgk", q, k.flatten(0, 1)) / math.sqrt(D)
            x = x.masked_fill(key[None, None] > last[:, None, None], -math.inf)
            total = x.logsumexp(-1)
            out[at, heads] = torch.einsum("tgk,kd->tgd", torch.exp(x - total[..., None]), v.flatten(0, 1))
            lse[at, heads] = total
    return out, lse


def exact(case, seed):
    """The outputs of run() in 64 bits; nothing where they are whole numbers, and where it would take long."""
    if case["op"] in ("extend", "select") or case["op"] == "append" and case["requests"] * case["q_hi"] > 200000:
        return None
    if case["op"] == "attention" and (work(case)["flops"] > 3e11 or
                                      len(_list_rows(case, _lengths(case)[0])[0]) * case["hkv"] > 8000):
        return None
    s = prepare(case, seed)
    return _exact_append(s, case) if case["op"] == "append" else _exact_attention(s, case)
