"""Oracle of the paged serving path (CPU, 64 bits, request after request). Test infrastructure only."""
import math

import torch

from .fp4 import quantize_nvfp4

PAGE = 128


def extend_pages(table, seq, new, free_pages, free_count, total_q, total_pages):
    """Every output of the operator as lists / tensors; the table is a copy."""
    table = table.clone()
    n, width = table.shape
    top, upto, status = max(0, min(int(free_count), free_pages.numel())), 0, 0
    left = top
    seq_out, cu_q, cu_k, cu_p, kv, slots = [], [0], [0], [0], [], []
    for r in range(n):
        o, m = max(int(seq[r]), 0), max(int(new[r]), 0)
        before, after = -(-o // PAGE), -(-(o + m) // PAGE)
        wide = after > width
        need = 0 if wide else after - before
        short = need > 0 and upto + need > top
        granted = not wide and not short
        status |= (1 if short else 0) | (2 if wide else 0)
        if granted:
            for i in range(need):
                table[r, before + i] = free_pages[top - 1 - (upto + i)]
            left = min(left, top - upto - need) if need else left
        upto += need
        k = o + m if granted else o
        seq_out.append(k)
        cu_q.append(cu_q[-1] + m)
        cu_k.append(cu_k[-1] + k)
        held = min(-(-k // PAGE), width)
        cu_p.append(cu_p[-1] + held)
        kv += table[r, :held].tolist()
        for i in range(m):
            p = o + i
            page = int(table[r, p // PAGE]) if granted else -1
            slots.append(page * PAGE + p % PAGE if page >= 0 else -1)
    status |= (4 if cu_q[-1] > total_q else 0) | (8 if cu_p[-1] > total_pages else 0)
    pad = lambda x, size: (x + [-1] * size)[:size]  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    cu_p = [min(x, total_pages) for x in cu_p]           # kv_indices has no more
    return dict(table=table, seq_lens=i32(seq_out), cu_seqlens_q=i32(cu_q), cu_seqlens_k=i32(cu_k), cu_page_offsets=i32(cu_p),
                kv_indices=i32(pad(kv, total_pages)), slots=torch.tensor(pad(slots, total_q), dtype=torch.int64),
                free_count=i32([left]), status=i32([status]))


def round_e4m3(x):
    """Nearest e4m3 value of a 64-bit x, ties to even, saturated; NaN stays."""
    e = torch.frexp(x)[1].sub(1).clamp(min=-6)
    step = torch.exp2((e - 3).double())
    return torch.where(torch.isnan(x), x, (torch.round(x / step) * step).clamp(-448, 448))


def append_tokens(codes, scale, x, cu_q, slots):
    """codes [P,H,128,128] and scale [P,H] (64 bits, copies) with the rows x [T,H,128] in."""
    codes, scale, x = codes.double().clone(), scale.double().clone(), x.double()
    for r in range(len(cu_q) - 1):
        t, end = int(cu_q[r]), int(cu_q[r + 1])
        if t < end and int(slots[t]) < 0:
            continue
        while t < end:
            page, o = divmod(int(slots[t]), PAGE)
            count = min(PAGE - o, end - t)
            rows = x[t:t + count].transpose(0, 1)
            top = torch.where(torch.isfinite(rows), rows.abs(), 0.0).amax((1, 2))
            need = torch.tensor([2.0 ** (-100 if a == 0 else max(-100, math.ceil(math.log2(a / 448)))) for a in top.tolist()],
                                dtype=torch.float64)
            if o:
                need = torch.maximum(need, scale[page])
                codes[page, :, :o] = round_e4m3(codes[page, :, :o] * (scale[page] / need)[:, None, None])
            scale[page] = need
            codes[page, :, o:o + count] = round_e4m3(rows / need[:, None, None])
            t += count
    return codes, scale


def append_index(k_index, k_index_scale, k, cu_q, slots):
    k_index, k_index_scale = k_index.clone(), k_index_scale.clone()
    packed, scales = quantize_nvfp4(k)
    for t in range(k.shape[0]):
        s = int(slots[t])
        if s >= 0:
            k_index[s // PAGE, :, s % PAGE] = packed[t]
            k_index_scale.view(torch.uint8)[s // PAGE, :, s % PAGE] = scales.view(torch.uint8)[t]
    return k_index, k_index_scale


def list_row(cu, r, i, tile):
    return cu + i if tile == 1 else cu // tile + r + i


def select_pages(scores, cu_q, seq, kv_heads, topk, tile=1, sink=1, recent=1, causal=True):
    hidx, pages, total = scores.shape
    n = len(cu_q) - 1
    rows = total if tile == 1 else total // tile + n
    ids = torch.full((kv_heads, rows, topk), -1, dtype=torch.int32)
    group = hidx // kv_heads
    for r in range(n):
        begin, end = int(cu_q[r]), int(cu_q[r + 1])
        for i in range(-(-(end - begin) // tile)):
            a, b = begin + i * tile, min(begin + (i + 1) * tile, end)
            seen = int(seq[r]) - (end - b) if causal else int(seq[r])
            seen = min(max(-(-seen // PAGE), 0), pages)
            for h in range(kv_heads):
                x = scores[h * group:(h + 1) * group, :, a:b].double()
                best = torch.where(torch.isnan(x), -math.inf, x).amax((0, 2)).tolist()
                order = []
                for p in range(seen):
                    if p < sink or p >= seen - recent:
                        order.append((0, 0.0, p))
                    elif best[p] > -math.inf:
                        order.append((1, -best[p], p))
                chosen = sorted(p for _, _, p in sorted(order)[:topk])
                ids[h, list_row(begin, r, i, tile), :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return ids


def paged_attention(q, k, v, k_scale, v_scale, table, seq, cu_q, ids=None, tile=1, causal=True, scale=None):
    """64-bit out [T,Hq,128], lse [T,Hq], the row's sum of p |v| (what the rounding of p scales with) and the largest
    scale * sum |q k| of its keys. Rows behind the last token are NaN."""
    total, hq, d = q.shape
    pages, hkv = k_scale.shape
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((total, hq, d), math.nan, dtype=torch.float64)
    lse = torch.full((total, hq), math.nan, dtype=torch.float64)
    spread, size = torch.zeros((total, hq, d), dtype=torch.float64), torch.zeros((total, hq), dtype=torch.float64)
    for r in range(len(cu_q) - 1):
        begin, end = int(cu_q[r]), min(int(cu_q[r + 1]), total)
        k_len = max(int(seq[r]), 0)
        held = min(-(-k_len // PAGE), table.shape[1])
        for t in range(begin, end):
            limit = k_len - (end - t) + 1 if causal else k_len
            for h in range(hkv):
                js = range(held) if ids is None else ids[h, list_row(begin, r, (t - begin) // tile, tile)].tolist()
                kk, vv = [], []
                for j in js:
                    if 0 <= j < held and j * PAGE < limit and 0 <= int(table[r, j]) < pages:
                        p, c = int(table[r, j]), min(limit - j * PAGE, PAGE)
                        kk.append(k[p, h, :c].double() * k_scale[p, h].double())
                        vv.append(v[p, h, :c].double() * v_scale[p, h].double())
                heads = slice(h * group, (h + 1) * group)
                if not kk:
                    out[t, heads], lse[t, heads] = 0.0, -math.inf
                    continue
                kk, vv = torch.cat(kk), torch.cat(vv)
                x = q[t, heads].double() @ kk.T * scale
                top = x.amax(-1, keepdim=True)
                dead = top == -math.inf
                p = torch.exp(x - torch.where(dead, 0.0, top))
                total_p = p.sum(-1, keepdim=True)
                p = torch.where(dead, 0.0, p / total_p)
                out[t, heads] = torch.where(dead, 0.0, p @ vv)
                lse[t, heads] = (top + total_p.log()).squeeze(-1)
                spread[t, heads] = p @ vv.abs()
                size[t, heads] = (q[t, heads].double().abs() @ kk.abs().T).amax(-1) * abs(scale)
    return out, lse, spread, size
