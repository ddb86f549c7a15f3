"""Serving over a paged 8-bit cache: page tables, cache writer, page lists and attention, bound to the C ABI.

extend_pages     lengths of a step -> pages from a free stack, block table, slot map, cumulative lengths, page list
append_tokens    bf16 keys and values -> e4m3 pages with a scale per (page, head), and NVFP4 index vectors
select_pages     scores of indexers.fp4_block_scores_varlen -> lists of pages
paged_attention  new tokens over all pages of their requests, or over listed ones
paged_step       all of them in order: one layer's step of a serving loop

A page holds 128 tokens, a head has 128 features. Rows of new tokens are packed request after request, `cu_seqlens_q`
[B + 1] gives their places. Everything runs on the current stream, nothing synchronises, and all entry points can be
captured in a CUDA graph after one eager call. No counterpart in the reference, whose ragged scorer
(indexers/fp4/vendor_minimax_msa/fp4_indexer_interface.py:745-811) reads a paged key cache that nothing else there uses."""
import collections
import contextlib
import ctypes
import functools
import math

import torch

from . import _lib
from .indexers import fp4_block_scores_varlen

PAGE = 128

# Arguments of the entry points: p a device pointer, q a 64-bit and i a 32-bit whole number, f an fp32, s the stream. With the
# types known to ctypes a call converts plain numbers, which is most of what a short call costs on the host.
_KINDS = dict(p=ctypes.c_void_p, q=ctypes.c_int64, i=ctypes.c_int, f=ctypes.c_float, s=ctypes.c_void_p)
_ENTRIES = dict(extend_pages="pqi" + "ppp" + "i" + "p" + "pppppppp" + "iii" + "s",
                append_tokens="pqq" + "pqq" + "pp" + "pppppp" + "iiiq" + "s",
                select_pages="pppp" + "iiiiiiiiii" + "s",
                paged_attention="pqq" + "pppp" + "pqi" + "ppp" + "ppp" + "q" + "iiii" + "q" + "iiii" + "f" + "s")


@functools.lru_cache(maxsize=None)
def _entry(name):
    fn = getattr(_lib.lib(), "sparse_b200_" + name)
    fn.argtypes = [_KINDS[k] for k in _ENTRIES[name]]
    fn.restype = ctypes.c_int
    return fn


def _on(device):
    """The device of a call made current, where it is not."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)

PageBatch = collections.namedtuple(
    "PageBatch", "seq_lens cu_seqlens_q cu_seqlens_k cu_page_offsets kv_indices slots free_count status")
STATUS_NO_PAGES, STATUS_TABLE_FULL, STATUS_TOKENS, STATUS_PAGES, STATUS_OVERFLOW = 1, 2, 4, 8, 16


def _bad(message):
    raise _lib.SparseB200Error(message)


def _dense(name, t, dtype, shape, device):
    if t.dtype is not dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        _bad(f"{name} must be a contiguous {dtype} tensor {list(shape)} on {device}")


def _rows(name, t, heads, device=None, total=None):
    """Packed bf16 rows [T, H, 128]: any token and head stride that keeps rows on 16 bytes."""
    shape = t.shape
    if t.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != 128 or not t.is_cuda:
        _bad(f"{name} must be a bfloat16 CUDA tensor [T,H,128]")
    if device is not None and t.device != device:
        _bad(f"{name} must be on {device}")
    if heads is not None and shape[1] != heads or total is not None and shape[0] != total:
        _bad(f"{name} must have shape [{total if total is not None else 'T'},{heads},128]")
    if t.requires_grad:
        _bad("the paged path is forward-only")
    (token, head, feature), at = t.stride(), t.data_ptr()
    if feature != 1 or (token | head) % 8 or at % 16:
        _bad(f"{name}: rows must be dense, 16-byte aligned and at strides that are multiples of 8 elements")
    return at, token, head


def _table(block_table, batch, device):
    """Its address, row stride and width."""
    shape, stride = block_table.shape, block_table.stride()
    if block_table.dtype is not torch.int32 or block_table.device != device or len(shape) != 2 or shape[0] != batch \
            or not 0 < shape[1] < 1 << 24 or stride[1] != 1 or batch > 1 and stride[0] < shape[1]:
        _bad("block_table must be int32 [B, pages per request] with dense rows on the same device")
    return block_table.data_ptr(), max(stride[0], shape[1]), shape[1]


class PagedCache:
    """Keys and values of one layer in pages of 128 tokens: e4m3 codes k, v [pages,Hkv,128,128] and scales k_scale, v_scale
    [pages,Hkv] fp32, and with index=True the NVFP4 index vectors of the keys, k_index [pages,Hkv,128,64] u8 and
    k_index_scale [pages,Hkv,128,8] e4m3, as fp4_block_scores_varlen takes them. Its tensors are the cache's own for good: they
    may be written to, not replaced (a cache over others is another from_tensors)."""

    _FIXED = frozenset(("k", "v", "k_scale", "v_scale", "k_index", "k_index_scale", "pages", "kv_heads", "device", "addresses"))

    def __setattr__(self, name, value):
        if name in self._FIXED:
            _bad(f"{name} of a cache cannot be replaced: use PagedCache.from_tensors")
        object.__setattr__(self, name, value)

    def __init__(self, pages, kv_heads, device="cuda", index=True):
        if pages <= 0 or kv_heads <= 0:
            _bad("pages and KV heads must be positive")
        shape = (pages, kv_heads, PAGE, 128)
        self._set(torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                  torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                  torch.ones(shape[:2], dtype=torch.float32, device=device),
                  torch.ones(shape[:2], dtype=torch.float32, device=device),
                  torch.zeros((*shape[:3], 64), dtype=torch.uint8, device=device) if index else None,
                  torch.zeros((*shape[:3], 8), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) if index else None)

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale, k_index=None, k_index_scale=None):
        """A cache over tensors that exist already (checked, not copied)."""
        cache = cls.__new__(cls)
        cache._set(k, v, k_scale, v_scale, k_index, k_index_scale)
        return cache

    def _set(self, k, v, k_scale, v_scale, k_index, k_index_scale):
        if k.dim() != 4 or tuple(k.shape[2:]) != (PAGE, 128) or not k.is_cuda:
            _bad("cache pages must be CUDA tensors [pages,Hkv,128,128]")
        pages, kv_heads = int(k.shape[0]), int(k.shape[1])
        lead = (pages, kv_heads)
        _dense("k", k, torch.float8_e4m3fn, (*lead, PAGE, 128), k.device)
        _dense("v", v, torch.float8_e4m3fn, (*lead, PAGE, 128), k.device)
        _dense("k_scale", k_scale, torch.float32, lead, k.device)
        _dense("v_scale", v_scale, torch.float32, lead, k.device)
        if (k_index is None) != (k_index_scale is None):
            _bad("index codes and scales go together")
        if k_index is not None:
            _dense("k_index", k_index, torch.uint8, (*lead, PAGE, 64), k.device)
            _dense("k_index_scale", k_index_scale, torch.float8_e4m3fn, (*lead, PAGE, 8), k.device)
        self.__dict__.update(k=k, v=v, k_scale=k_scale, v_scale=v_scale, k_index=k_index, k_index_scale=k_index_scale, pages=pages,
                             kv_heads=kv_heads, device=k.device)

    @property
    def addresses(self):
        """Of codes, scales and index vectors (0: none), as they are at the time of a call."""
        at = self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()
        return (*at, 0, 0) if self.k_index is None else (*at, self.k_index.data_ptr(), self.k_index_scale.data_ptr())


def extend_pages(block_table, seq_lens, new_lens, free_pages, free_count, *, total_q, total_pages):
    """Pages for new_lens [B] tokens behind the seq_lens [B] that the requests hold, taken from the end of free_pages
    [free_count], and the tables of the step. block_table [B, W] is extended in place; everything else is new (PageBatch):
    seq_lens with the new tokens, cu_seqlens_q / cu_seqlens_k / cu_page_offsets [B+1], kv_indices [total_pages], slots
    [total_q] int64, free_count [1], status [1] (STATUS_* bits; 0: all is well). total_q and total_pages are the sizes of the
    tables; what is behind the last token or page is -1, and cu_page_offsets never goes beyond total_pages (STATUS_PAGES says
    that pages were left out). A request that gets no pages is refused: its length stays, its slots are -1, and what a step
    gives for its rows means nothing."""
    batch, dev = seq_lens.numel(), seq_lens.device
    if not seq_lens.is_cuda or batch == 0:
        _bad("seq_lens must be a CUDA tensor of at least one request")
    _dense("seq_lens", seq_lens, torch.int32, (batch,), dev)
    _dense("new_lens", new_lens, torch.int32, (batch,), dev)
    _dense("free_pages", free_pages, torch.int32, (free_pages.numel(),), dev)
    _dense("free_count", free_count, torch.int32, (1,), dev)
    table, stride, width = _table(block_table, batch, dev)
    if not 0 <= total_q < 1 << 31 or not 0 <= total_pages < 1 << 31:
        _bad("table sizes must not be negative, and fit int32")
    with _on(dev):
        # one allocation, the 64-bit slots first
        buffer = torch.empty(2 * total_q + 4 * batch + 5 + total_pages, dtype=torch.int32, device=dev)
        slots, seq, cu_q, cu_k, cu_pages, count, status, kv = torch.unsafe_split_with_sizes(
            buffer, (2 * total_q, batch, batch + 1, batch + 1, batch + 1, 1, 1, total_pages))
        at_slots, step = buffer.data_ptr(), 4 * batch + 4
        at = at_slots + 8 * total_q
        at_q = at + 4 * batch
        at_count = at_q + 3 * step
        _lib.check(_entry("extend_pages")(
            table, stride, width, seq_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(), free_pages.numel(),
            free_count.data_ptr(), at, at_q, at_q + step, at_q + 2 * step, at_count + 8, at_slots, at_count, at_count + 4,
            batch, total_q, total_pages, _stream(dev)))
    return PageBatch(seq, cu_q, cu_k, cu_pages, kv, slots.view(torch.int64), count, status)


def append_tokens(cache, k, v, cu_seqlens_q, slots):
    """k, v [T,Hkv,128] bf16 -> the rows of the cache that slots [T] (extend_pages) names: the tokens of a request lie in
    order from its first slot, page after page. A page's scale is the smallest power of two that holds its rows; the rows
    before the new ones are rescaled where it grows. Index vectors are written where the cache has them."""
    total, dev = slots.numel(), cache.device
    rows = (*_rows("k", k, cache.kv_heads, dev, total), *_rows("v", v, cache.kv_heads, dev, total))
    batch = cu_seqlens_q.numel() - 1
    _dense("cu_seqlens_q", cu_seqlens_q, torch.int32, (batch + 1,), dev)
    _dense("slots", slots, torch.int64, (total,), dev)
    with _on(dev):
        _lib.check(_entry("append_tokens")(*rows, cu_seqlens_q.data_ptr(), slots.data_ptr(), *cache.addresses, batch,
                                           cache.kv_heads, total, cache.pages, _stream(dev)))


def list_rows(total_q, batch, tile):
    """Rows of the lists of a step: tile i of request r has row cu_seqlens_q[r] // tile + r + i (tile 1: the token's row)."""
    return total_q if tile == 1 else total_q // tile + batch


MOST_PAGES = 51199          # of a request whose pages select_pages takes


def _check_selection(pages, kv_heads, topk, tile, sink, recent):
    if tile < 1 or tile > 128 or tile & (tile - 1) or kv_heads < 1 or topk < 1:
        _bad("tile must be a power of two from 1 to 128, KV heads and topk positive")
    if sink < 0 or recent < 0 or sink + recent > topk:
        _bad("sink and recent pages must fit the list")
    if pages < 1 or pages > MOST_PAGES:
        _bad(f"the page selection takes 1 to {MOST_PAGES} pages of a request")


def select_pages(scores, cu_seqlens_q, seq_lens, *, kv_heads, topk, tile=1, sink=1, recent=1, causal=True, ids=None):
    """scores [Hidx, pages, T] fp32 (fp4_block_scores_varlen) -> ids [kv_heads, list_rows(T, B, tile), topk] int32: for every
    `tile` consecutive tokens of a request the best pages by (score descending, page ascending), written ascending with -1
    behind them. The first `sink` and the last `recent` pages that the tile's last token sees are always among them."""
    if not scores.is_cuda or scores.dtype is not torch.float32 or scores.dim() != 3 or not scores.is_contiguous():
        _bad("scores must be contiguous float32 [Hidx,pages,T] on CUDA")
    hidx, pages, total = scores.shape
    dev, batch = scores.device, seq_lens.numel()
    _dense("seq_lens", seq_lens, torch.int32, (batch,), dev)
    _dense("cu_seqlens_q", cu_seqlens_q, torch.int32, (batch + 1,), dev)
    _check_selection(pages, kv_heads, topk, tile, sink, recent)
    shape = (kv_heads, list_rows(total, batch, tile), topk)
    with _on(dev):
        if ids is None:
            ids = torch.empty(shape, dtype=torch.int32, device=dev)
        else:
            _dense("ids", ids, torch.int32, shape, dev)
        _lib.check(_entry("select_pages")(
            scores.data_ptr(), cu_seqlens_q.data_ptr(), seq_lens.data_ptr(), ids.data_ptr(), batch, hidx, kv_heads, pages, total,
            topk, tile, sink, recent, bool(causal), _stream(dev)))
    return ids


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device, hq, hkv, tile, max_q, listed):
    fn = _lib.lib().sparse_b200_paged_attention_workspace_bytes
    fn.restype = ctypes.c_int64
    with torch.cuda.device(device):
        n = fn(hq, hkv, tile, max_q, listed)
    if n < 0:
        _lib.check(n)
    return n


def _check_queries(q, cache):
    """Tokens, query heads, and the rows' address and strides."""
    rows, hkv = _rows("q", q, None, cache.device), cache.kv_heads
    total, hq, _ = q.shape
    if hq < hkv or hq % hkv or hq // hkv > 64:
        _bad("Hq must be a multiple of Hkv, at most 64 query heads to a KV head")
    return total, hq, rows


def paged_attention(q, cache, block_table, seq_lens, cu_seqlens_q, ids=None, *, tile=1, max_seqlen_q=None, causal=True,
                    scale=None, out=None, lse=None, return_lse=False):
    """softmax(scale q k^T) v of q [T,Hq,128] bf16 over the pages of each request (ids=None) or the listed ones (ids
    [Hkv, list_rows(T, B, tile), topk] of select_pages). seq_lens [B] count the new tokens in; causal: token i of n sees the
    keys j <= i + seq_len - n. Returns out [T,Hq,128] bf16, with return_lse also the natural-log LSE [T,Hq] fp32; rows behind
    the last token of out and lse are left as they were. max_seqlen_q: the largest number of new tokens, for how many of them
    share a pass over a page (default: T). scale: default 128^-0.5."""
    hkv, dev, batch = cache.kv_heads, cache.device, seq_lens.numel()
    total, hq, rows = _check_queries(q, cache)
    _dense("seq_lens", seq_lens, torch.int32, (batch,), dev)
    _dense("cu_seqlens_q", cu_seqlens_q, torch.int32, (batch + 1,), dev)
    table = _table(block_table, batch, dev)
    topk = 0
    if ids is not None:
        if ids.dim() != 3 or ids.shape[2] < 1 or tile < 1 or tile > 128 or tile & (tile - 1):
            _bad("ids must be [Hkv, list rows, topk] for a tile that is a power of two from 1 to 128")
        topk = ids.shape[2]
        _dense("ids", ids, torch.int32, (hkv, list_rows(total, batch, tile), topk), dev)
    max_q = total if max_seqlen_q is None else int(max_seqlen_q)
    with _on(dev):
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty((total, hq, 128), dtype=torch.bfloat16, device=dev)
        else:
            _dense("out", out, torch.bfloat16, (total, hq, 128), dev)
            for t in (q, cache.k, cache.v):
                if out.untyped_storage().data_ptr() == t.untyped_storage().data_ptr():
                    _bad("output must not alias inputs")
        if lse is not None:
            _dense("lse", lse, torch.float32, (total, hq), dev)
        elif return_lse:
            lse = torch.empty((total, hq), dtype=torch.float32, device=dev)
        # scratch of this call alone, from torch's caching allocator (inside torch.cuda.graph it belongs to the graph)
        need = _workspace_bytes(dev.index, hq, hkv, tile, max_q, topk > 0)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(_entry("paged_attention")(
            *rows, *cache.addresses[:4], *table, seq_lens.data_ptr(), cu_seqlens_q.data_ptr(),
            0 if ids is None else ids.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), ws.data_ptr(), need, batch,
            hq, hkv, total, cache.pages, topk, tile, max_q, bool(causal), 128 ** -0.5 if scale is None else scale, _stream(dev)))
    return (out, lse) if return_lse else out


def paged_step(q, k, v, cache, block_table, batch, *, topk=None, tile=1, max_seqlen_q, max_seqlen_k, sink=1, recent=1,
               scale=None):
    """One layer's step over a PageBatch: append k, v to the cache, score the pages of every request with the NVFP4 index
    vectors (one index head per KV head: the mean of its query heads), select topk of them and attend. topk=None: attend to
    whole sequences, without index vectors. Returns (out, ids); rows whose slot is -1 (a refused request's, and those behind the
    last token) have no meaning."""
    # what a later stage would refuse is refused before the cache has changed
    tokens, dev, requests = _check_queries(q, cache)[0], cache.device, batch.seq_lens.numel()
    _table(block_table, requests, dev)
    _dense("seq_lens", batch.seq_lens, torch.int32, (requests,), dev)
    _dense("cu_seqlens_q", batch.cu_seqlens_q, torch.int32, (requests + 1,), dev)
    if scale is not None and not abs(scale) < 2.0 ** 128 - 2.0 ** 103:        # fp32, rounded
        _bad("scale must be finite")
    if cache.pages * cache.kv_heads * PAGE >= 1 << 31:
        _bad("rows of the cache must fit int32")
    if topk is not None:
        if cache.k_index is None:
            _bad("selection needs a cache with index vectors")
        _dense("cu_seqlens_k", batch.cu_seqlens_k, torch.int32, (requests + 1,), dev)
        _dense("cu_page_offsets", batch.cu_page_offsets, torch.int32, (requests + 1,), dev)
        _dense("kv_indices", batch.kv_indices, torch.int32, (batch.kv_indices.numel(),), dev)
        if tokens and (max_seqlen_q < 1 or max_seqlen_k < 1 or batch.kv_indices.numel() == 0):
            _bad("lengths and the page list of a step with tokens must not be empty")
        _check_selection(max((max_seqlen_k + PAGE - 1) // PAGE, 1), cache.kv_heads, topk, tile, sink, recent)
    append_tokens(cache, k, v, batch.cu_seqlens_q, batch.slots)
    ids = None
    if topk is not None:
        if tokens:
            codes, scales = quantize_rows(q, cache.kv_heads)
            scores = fp4_block_scores_varlen(codes, cache.k_index, scales, cache.k_index_scale, batch.cu_seqlens_q,
                                             batch.cu_seqlens_k, batch.cu_page_offsets, max_seqlen_q=max_seqlen_q,
                                             max_seqlen_k=max_seqlen_k, kv_indices=batch.kv_indices, causal=True, exact=False)
        else:
            scores = torch.empty((cache.kv_heads, 1, 0), dtype=torch.float32, device=dev)
        ids = select_pages(scores, batch.cu_seqlens_q, batch.seq_lens, kv_heads=cache.kv_heads, topk=topk, tile=tile,
                           sink=sink, recent=recent)
    out = paged_attention(q, cache, block_table, batch.seq_lens, batch.cu_seqlens_q, ids, tile=tile,
                          max_seqlen_q=max_seqlen_q, scale=scale)
    return out, ids


def quantize_rows(q, hidx):
    """Packed rows q [T,Hq,128] bf16 (strides as everywhere here; rows that are not contiguous are copied first) -> NVFP4 query
    index vectors (codes [T,hidx,64], scales [T,hidx,8]): the mean over the Hq/hidx heads of a group, as
    indexers.quantize_queries for whole sequences."""
    _rows("q", q, None)
    total, hq = q.shape[:2]
    if hidx < 1 or hq % hidx or hq < hidx:
        _bad("Hq must be a multiple of the index head count")
    with _on(q.device):
        codes = torch.empty((total, hidx, 64), dtype=torch.uint8, device=q.device)
        scales = torch.empty((total, hidx, 8), dtype=torch.float8_e4m3fn, device=q.device)
        if total:      # T batches of one token
            q = q.contiguous()
            _lib.check(_lib.lib().sparse_b200_nvfp4_quantize(_lib.ptr(q), _lib.ptr(codes), _lib.ptr(scales), total, hidx,
                                                             hq // hidx, 1, 0, ctypes.c_void_p(_stream(q.device))))
    return codes, scales
