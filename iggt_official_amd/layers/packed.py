"""Attention over packed sequences of different lengths, and over K/V that stay between calls in an 8-bit paged cache.

The reference runs a scene whole: equal-length batches through F.scaled_dot_product_attention (iggt/layers/attention.py:60-66).
These operators serve what it has no form for -- scenes of different numbers of views in one call, and a scene that grows view by
view (or token by token) against everything it has seen:

    packed_attention   causal or full attention, grouped heads, over packed rows
    plan_pages         block tables and slot maps from request lengths, on the GPU
    append_pages       writes new K/V rows into the cache: e4m3 codes, one power-of-two scale per page and key head
    paged_attention    attention of new rows (one or many per request) over the cache
    PagedKVCache       the buffers of the last three, and calls that go together

Forward only (no autograd history: inputs that require gradients are refused while gradients are recorded).  Calls enqueue on the
current stream of the tensors' device and do not wait; scratch comes from torch's allocator per call, so captured graphs do not
share it.  Index tensors (lengths, prefix sums, tables, slots) are device data and are not read back: the kernels clamp them to the
tensors they index.
"""
import functools
import struct
from typing import NamedTuple, Optional

import torch

from .. import _C

_INT, _BYTE = torch.int32, torch.uint8
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
MAX_REQUESTS = 8192
MAX_ROWS = 2 ** 31 - 2 ** 20     # rows, keys, planned slots of a call: 32-bit numbers below the Python API


# Calls of a few microseconds: conditions first, messages only where one fails, and no object that a plain number can stand for.
_current, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


# iggt_seq_call: a word that names the call and its arguments, 8 bytes each (ctypes converts thirty arguments in 2.7 us, struct in 0.3)
_PACKED, _PAGED, _APPEND, _PLAN = (struct.Struct(f) for f in ("=23qd4q", "=25qd4q", "=18q", "=17q"))
_CALL = {_PACKED: "iggt_packed_attn", _PAGED: "iggt_paged_attn", _APPEND: "iggt_append_pages", _PLAN: "iggt_plan_pages"}
_PACKED_BF16, _PAGED_BF16, _APPEND_BF16, _PLAN_PAGES = 0, 2, 4, 6     # fp16: one more


def _call(layout, *words):
    rc = _C.load().iggt_seq_call(layout.pack(*words))
    if rc:
        _C._check(rc, _CALL[layout])


def _refuse(what):
    raise _C.HipExtensionError(what)


def _strides(name, t, step):
    """(address, row stride, head stride) of a [rows, heads, channels] operand; dimensions of one entry have no stride."""
    rs, hs, cs = t.stride()
    at = t.data_ptr()
    if cs != 1 or (rs | hs) % step or at % (2 * step):
        rows, heads, _ = t.shape
        rs, hs = (0 if rows <= 1 else rs), (0 if heads == 1 else hs)
        if cs != 1 or (rs | hs) % step or at % (2 * step):
            _refuse(f"{name}: channels have to be contiguous, strides multiples of {step} elements and the start aligned to {2 * step} bytes")
    return at, rs, hs


def _query(q, out, grad):
    """Checks of the query rows and of the output that hold for both attentions; returns the output."""
    if q.dim() != 3 or q.dtype not in _C.H16 or q.shape[2] not in HEAD_DIMS:
        _refuse(f"q: bf16 or fp16 [rows, heads, 64 | 128] expected, got {q.dtype} {tuple(q.shape)}")
    if grad and torch.is_grad_enabled():
        _refuse("packed / paged attention is forward only: an input requires gradients")
    if q.shape[0] * q.shape[1] >= MAX_ROWS:
        _refuse(f"{q.shape[0]} x {q.shape[1]} query rows and heads are more than {MAX_ROWS}")
    if out is None:
        return torch.zeros_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != q.get_device():
        _refuse("out has to have q's shape, type and device")
    if out.requires_grad and torch.is_grad_enabled():
        _refuse("packed / paged attention is forward only: out requires gradients")
    rs, hs, _ = out.stride()
    if (rs == 0 and q.shape[0] > 1) or (hs == 0 and q.shape[1] > 1):
        _refuse("out is an expanded view")
    return out


def _index(name, t, n, where):
    """Address of a contiguous int32 [n] on device number `where`."""
    if t.dtype != _INT or t.shape != (n,) or t.get_device() != where or not t.is_contiguous():
        _refuse(f"{name}: contiguous int32 [{n}] on cuda:{where} expected, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    scale = float(scale)
    if not 1e-37 <= scale <= 1e37:      # (a float32 below)
        _refuse(f"softmax scale has to be positive and between 1e-37 and 1e37, got {scale}")
    return scale


@functools.lru_cache(maxsize=1024)
def _ws_bytes(name, *sizes):
    return int(getattr(_C.load(), name)(*sizes))


def packed_attention(q, k, v, cu_q, cu_k, max_q: int, max_k: int, *, causal: bool = True, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None):
    """softmax(scale q k^T) v within every sequence: rows cu_q[b] .. cu_q[b + 1] of q [Tq, Hq, D] over keys cu_k[b] .. cu_k[b + 1] of
    k, v [Tk, Hkv, D] (bf16 or fp16, D 64 | 128, Hq a multiple of Hkv; query head h reads key head h // (Hq // Hkv)).  causal: row i of
    Lq sees keys j <= i + Lk - Lq; a row that sees none (or only scores of -inf) is 0.  scale: default D ** -0.5.

    max_q, max_k: the longest sequences' lengths or more (of a sequence with more rows the first max_q are computed, as they would be
    with all of them; max_k only steers how the work is split).  out: rows that belong to no sequence are left as they are; without it
    they are 0.  It may be q itself, and must not overlap q in another way, nor k or v.  Rows of k and of v lie less than 2^24 elements
    apart.  Prefix sums do not decrease: a row that two sequences share has the values of either."""
    where = q.get_device()
    if where < 0:
        _refuse("IGGT HIP ops need tensors on a ROCm device (no CPU fallback)")
    if where != _current():
        with torch.cuda.device(where):
            return packed_attention(q, k, v, cu_q, cu_k, max_q, max_k, causal=causal, scale=scale, out=out)
    out = _query(q, out, q.requires_grad or k.requires_grad or v.requires_grad)
    dtype, kv = q.dtype, k.shape
    tq, hq, dim = q.shape
    if len(kv) != 3 or kv != v.shape or kv[2] != dim or k.dtype != dtype or v.dtype != dtype or k.get_device() != where or v.get_device() != where:
        _refuse(f"k, v: {dtype} [keys, heads, {dim}] on {q.device} expected, got {k.dtype} {tuple(kv)} on {k.device} and {v.dtype} {tuple(v.shape)} on {v.device}")
    tk, hkv, _ = kv
    if hkv == 0 or hq == 0 or hq % hkv:
        _refuse(f"{hq} query heads are no multiple of {hkv} key heads")
    batch = cu_q.numel() - 1
    if not 0 <= batch < MAX_ROWS or tk >= MAX_ROWS:
        _refuse(f"cu_q: one entry more than there are sequences expected; fewer than {MAX_ROWS} sequences and keys")
    starts = _index("cu_q", cu_q, batch + 1, where), _index("cu_k", cu_k, batch + 1, where)
    max_q, max_k = min(int(max_q), tq), min(int(max_k), tk)
    if max_q < 0 or max_k < 0:
        _refuse("max_q and max_k are lengths")
    scale = _scale(scale, dim)
    rows = *_strides("q", q, 8), *_strides("k", k, 8), *_strides("v", v, 8), *_strides("out", out, 4)
    if batch == 0 or max_q == 0:
        return out
    n = _ws_bytes("iggt_packed_attn_ws_bytes", batch, max_q, max_k, hq, hkv, dim)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _call(_PACKED, _PACKED_BF16 + (dtype == torch.float16), *rows, *starts, batch, tq, tk, max_q, max_k, hq, hkv, dim, scale,
          1 if causal else 0, ws.data_ptr() if n else 0, n, _stream(where))
    return out


class Pages(NamedTuple):
    """Buffers of the cache, uint8: K codes [pages, key heads, page, D], V codes [pages, key heads, page / 16, D, 16] (e4m3 bytes; 16
    tokens of a V channel lie side by side), scale exponents [pages, key heads] (a code c stands for c * 2 ** (byte - 127))."""
    k_codes: torch.Tensor
    k_scale: torch.Tensor
    v_codes: torch.Tensor
    v_scale: torch.Tensor

    @staticmethod
    def empty(pages: int, kv_heads: int, head_dim: int, page: int = 64, device="cuda") -> "Pages":
        if page not in PAGE_SIZES or head_dim not in HEAD_DIMS or pages < 0 or kv_heads <= 0:
            _refuse(f"pages of {PAGE_SIZES} tokens and head dims {HEAD_DIMS} expected, got {page} and {head_dim}")
        make = functools.partial(torch.zeros, dtype=torch.uint8, device=device)
        return Pages(make(pages, kv_heads, page, head_dim), make(pages, kv_heads), make(pages, kv_heads, page // 16, head_dim, 16),
                     make(pages, kv_heads))


def _pages(pages, where):
    """(number of pages, key heads, page size, head dim) of a checked cache."""
    k, ks, v, vs = pages
    n, heads, page, dim = k.shape if k.dim() == 4 else (0, 0, 0, 0)
    if page not in PAGE_SIZES or dim not in HEAD_DIMS or heads == 0 or n * page >= 2 ** 31:
        _refuse(f"K codes: [pages, heads, {PAGE_SIZES}, {HEAD_DIMS}] expected, got {tuple(k.shape)}")
    if ks.shape != (n, heads) or vs.shape != (n, heads) or v.shape != (n, heads, page // 16, dim, 16):
        _refuse(f"cache buffers do not belong together: {[tuple(t.shape) for t in pages]}")
    for t in pages:
        if t.dtype != _BYTE or t.get_device() != where or not t.is_contiguous():
            _refuse(f"cache buffers: contiguous uint8 on cuda:{where} expected, got {t.dtype} on {t.device}")
    return n, heads, page, dim


def append_pages(pages: Pages, k, v, slots):
    """Writes k, v [T, key heads, D] (bf16 or fp16) into the cache at slots [T] (int32: page * page size + place; rows whose slot is
    not in the cache are skipped).  Rows of one page have to be one run of consecutive slots, as plan_pages gives them: a page that
    appears in two runs of one call has no defined content.  The scale of a page is the least power of two that holds its largest
    finite value, and never falls while the page is being filled; held codes are rewritten when it grows."""
    where = k.get_device()
    if where < 0:
        _refuse("IGGT HIP ops need tensors on a ROCm device (no CPU fallback)")
    if where != _current():
        with torch.cuda.device(where):
            return append_pages(pages, k, v, slots)
    dtype = k.dtype
    n, heads, page, dim = _pages(pages, where)
    if k.dim() != 3 or k.shape[1:] != (heads, dim) or dtype not in _C.H16 or v.shape != k.shape or v.dtype != dtype or v.get_device() != where:
        _refuse(f"k, v: bf16 or fp16 [tokens, {heads}, {dim}] of one type expected, got {tuple(k.shape)} {dtype} and {tuple(v.shape)} {v.dtype}")
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        _refuse("append_pages is forward only: an input requires gradients")
    tokens = k.shape[0]
    if tokens >= 2 ** 30:
        _refuse(f"fewer than 2^30 tokens expected, got {tokens}")
    _call(_APPEND, _APPEND_BF16 + (dtype == torch.float16), *_strides("k", k, 8), *_strides("v", v, 8),
          _index("slots", slots, tokens, where), tokens, pages.k_codes.data_ptr(), pages.k_scale.data_ptr(), pages.v_codes.data_ptr(),
          pages.v_scale.data_ptr(), n, page, heads, dim, _stream(where))
    return pages


def paged_attention(q, pages: Pages, tables, lens, max_q: int, max_len: int, *, cu_q=None, causal: bool = True,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None):
    """packed_attention's formula with keys and values out of the cache: request b's token t is place t % page of page
    tables[b, t // page], and it holds lens[b] of them (the new ones among them).  q [Tq, Hq, D]: rows cu_q[b] .. cu_q[b + 1] of request b
    are its last tokens; cu_q None: one row per request, row b.  causal: row i of Lq sees tokens t <= i + lens[b] - Lq.

    max_q, max_len: the largest number of rows, of tokens, or more (as max_q and max_k there).  Tokens on a page that does not exist
    count as not there.  out: as in packed_attention.  fp16 rows: cached V beyond 131 008 in magnitude (written from bf16) is infinite."""
    where = q.get_device()
    if where < 0:
        _refuse("IGGT HIP ops need tensors on a ROCm device (no CPU fallback)")
    if where != _current():
        with torch.cuda.device(where):
            return paged_attention(q, pages, tables, lens, max_q, max_len, cu_q=cu_q, causal=causal, scale=scale, out=out)
    out = _query(q, out, q.requires_grad)
    dtype = q.dtype
    tq, hq, dim = q.shape
    n, hkv, page, d = _pages(pages, where)
    if d != dim or hq == 0 or hq % hkv:
        _refuse(f"q has {hq} heads of {dim}, the cache {hkv} of {d}")
    batch, width, stride = _tables(tables, where, page)
    if batch >= MAX_ROWS:
        _refuse(f"fewer than {MAX_ROWS} requests expected")
    held = _index("lens", lens, batch, where)
    max_q, max_len = min(int(max_q), tq), min(int(max_len), width * page)
    if max_q < 0 or max_len < 0:
        _refuse("max_q and max_len are lengths")
    starts = 0
    if cu_q is not None:
        starts = _index("cu_q", cu_q, batch + 1, where)
    elif max_q > 1 or tq < batch:
        _refuse("without cu_q there is one row per request")
    scale = _scale(scale, dim)
    rows = *_strides("q", q, 8), *_strides("out", out, 4)
    if batch == 0 or max_q == 0:
        return out
    nbytes = _ws_bytes("iggt_paged_attn_ws_bytes", batch, max_q, max_len, hq, hkv, dim)
    ws = torch.empty(nbytes, dtype=_BYTE, device=q.device) if nbytes else None
    _call(_PAGED, _PAGED_BF16 + (dtype == torch.float16), *rows, pages.k_codes.data_ptr(), pages.k_scale.data_ptr(),
          pages.v_codes.data_ptr(), pages.v_scale.data_ptr(), n, page, tables.data_ptr(), stride, width, held, starts, batch, tq, max_q,
          max_len, hq, hkv, dim, scale, 1 if causal else 0, ws.data_ptr() if nbytes else 0, nbytes, _stream(where))
    return out


def _tables(tables, where, page):
    """(requests, width, row stride) of checked block tables."""
    if tables.dim() != 2 or tables.dtype != _INT or tables.get_device() != where:
        _refuse(f"tables: int32 [requests, pages of the longest] on cuda:{where} expected, got {tables.dtype} {tuple(tables.shape)} on {tables.device}")
    requests, width = tables.shape
    rs, cs = tables.stride()
    if (width > 1 and cs != 1) or (requests > 1 and rs < width):
        _refuse("tables: contiguous rows that do not overlap expected")
    if width * page >= 2 ** 31 - 1024:
        _refuse("more than 2^31 slots")
    return requests, width, rs


def plan_pages(tables, ring, counters, lens, new_lens, page: int, tokens: int):
    """One step of the block tables: requests that hold lens [R] tokens are to hold new_lens [R] (more: tokens are appended; fewer: the
    last ones are dropped; 0: the request ends).  Growing requests take pages from the head of `ring` [N] (free pages ring[(head + i) % N],
    i < count; counters = (head, count, ...)), pages no longer needed go behind its tail for later steps, both in request order.  Pages are
    numbered 0 .. N - 1 (a token on any other has slot -1).  tables [R, width] and ring are updated in place; lens and counters are not.

    Returns (tables, ring, starts [R + 1], next_lens [R], next_counters [3] = (head, count, missing), slots [tokens]): slots of the
    added tokens in request order, -1 behind the last, request b's at starts[b] .. starts[b + 1].  `missing` pages > 0 (or -1: `tokens` is
    too small) means that no request has grown in this step."""
    where = tables.get_device()
    if where < 0:
        _refuse("IGGT HIP ops need tensors on a ROCm device (no CPU fallback)")
    if where != _current():
        with torch.cuda.device(where):
            return plan_pages(tables, ring, counters, lens, new_lens, page, tokens)
    if page not in PAGE_SIZES:
        _refuse(f"pages hold {PAGE_SIZES} tokens, not {page}")
    requests, width, stride = _tables(tables, where, page)
    tokens, size = int(tokens), ring.numel()
    if requests > MAX_REQUESTS or requests * width >= 2 ** 31 or not 0 <= tokens < MAX_ROWS or size * page >= 2 ** 31:
        _refuse(f"at most {MAX_REQUESTS} requests, fewer than 2^31 table entries and slots and {MAX_ROWS} new tokens expected")
    if counters.numel() < 2:
        _refuse("counters: int32 (head, count, ...) expected")
    inputs = (_index("counters", counters, counters.numel(), where), _index("lens", lens, requests, where),
              _index("new_lens", new_lens, requests, where))
    free = _index("ring", ring, size, where)
    buf = torch.empty(2 * requests + 4 + tokens, dtype=_INT, device=tables.device)     # one allocation for the four outputs
    starts, next_lens, next_counters, slots = torch.unsafe_split_with_sizes(buf, (requests + 1, requests, 3, tokens))
    at = buf.data_ptr()
    _call(_PLAN, _PLAN_PAGES, tables.data_ptr(), stride, requests, width, free, size, *inputs, page, at, at + 4 * (requests + 1),
          at + 4 * (2 * requests + 1), at + 4 * (2 * requests + 4), tokens, _stream(where))
    return tables, ring, starts, next_lens, next_counters, slots


class PagedKVCache:
    """K/V of up to `requests` requests in `pages` pages of `page` tokens.  A step: plan -> append -> attend.

        cache = PagedKVCache(requests=4, longest=65536, pages=1024, kv_heads=16, head_dim=64)
        starts, slots = cache.plan(new_lens, tokens=k.shape[0])      # int32 [4]: tokens each request holds after the step
        cache.append(k, v, slots)                                     # rows of the added tokens, request by request
        o = cache.attend(q, max_q, max_len, cu_q=starts)              # q: the added tokens' rows

    `lens` [requests] and `counters` (head, free pages, pages missing in the last step) are updated in place, so a captured graph of
    a step goes on where the last replay ended."""

    def __init__(self, requests: int, longest: int, pages: int, kv_heads: int, head_dim: int, page: int = 64, device="cuda"):
        if not 0 < requests <= MAX_REQUESTS or longest <= 0 or pages <= 0:
            _refuse(f"up to {MAX_REQUESTS} requests, of one token or more, and one page or more expected")
        self.page = page
        self.pages = Pages.empty(pages, kv_heads, head_dim, page, device)
        device = self.pages.k_codes.device
        self.tables = torch.full((requests, -(-longest // page)), -1, dtype=_INT, device=device)
        self.ring = torch.arange(pages, dtype=_INT, device=device)
        self.counters = torch.tensor([0, pages, 0], dtype=_INT, device=device)
        self.lens = torch.zeros(requests, dtype=_INT, device=device)

    def plan(self, new_lens, tokens: int):
        """(starts, slots) of the step that takes every request to new_lens tokens, of which `tokens` at most are added in all."""
        _, _, starts, lens, counters, slots = plan_pages(self.tables, self.ring, self.counters, self.lens, new_lens, self.page, tokens)
        self.lens.copy_(lens), self.counters.copy_(counters)
        return starts, slots

    def append(self, k, v, slots):
        append_pages(self.pages, k, v, slots)

    def attend(self, q, max_q: int, max_len: int, *, cu_q=None, causal: bool = True, scale: Optional[float] = None, out=None):
        return paged_attention(q, self.pages, self.tables, self.lens, max_q, max_len, cu_q=cu_q, causal=causal, scale=scale, out=out)
