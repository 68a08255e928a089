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
from typing import NamedTuple, Optional

import torch

from .. import _C

_INT = torch.int32
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
MAX_REQUESTS = 8192


def _need(ok, what):
    if not ok:
        raise _C.HipExtensionError(what)


def _call(name, device, *args):
    """C entry on the current stream of `device`, whichever device is current."""
    fn = getattr(_C.load(), name)
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    _C._check(rc, name)


def _strides(name, t, step):
    """(row, head) strides of a [rows, heads, channels] operand; dimensions of one entry have none."""
    rows, heads, dim = t.shape
    rs, hs, cs = t.stride()
    rs, hs = (0 if rows <= 1 else rs), (0 if heads == 1 else hs)
    _need(cs == 1 and rs % step == 0 and hs % step == 0 and t.data_ptr() % (2 * step) == 0,
          f"{name}: channels have to be contiguous, strides multiples of {step} elements and the start aligned to {2 * step} bytes")
    return rs, hs


def _operands(q, out, **others):
    """Checks that hold for both attentions; returns the output."""
    _need(q.is_cuda, "IGGT HIP ops need tensors on a ROCm device (no CPU fallback)")
    _need(q.dim() == 3 and q.dtype in _C.H16 and q.shape[2] in HEAD_DIMS, f"q: bf16 or fp16 [rows, heads, 64 | 128] expected, got {q.dtype} {tuple(q.shape)}")
    grad = q.requires_grad
    for name, t in others.items():
        _need(t.device == q.device, f"{name} is on {t.device}, q on {q.device}")
        grad = grad or t.requires_grad
    _need(not (grad and torch.is_grad_enabled()), "packed / paged attention is forward only: an input requires gradients")
    if out is None:
        return torch.zeros_like(q, memory_format=torch.contiguous_format)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out has to have q's shape, type and device")
    _need(all(n == 1 or s > 0 for n, s in zip(out.shape, out.stride())), "out is an expanded view")
    return out


def _index(name, t, shape, device):
    _need(t.dtype == _INT and t.device == device and tuple(t.shape) == shape and t.is_contiguous(),
          f"{name}: contiguous int32 {list(shape)} on {device} expected, got {t.dtype} {list(t.shape)} on {t.device}")


def _scale(scale, dim):
    scale = dim ** -0.5 if scale is None else float(scale)
    _need(0.0 < scale < float("inf"), f"softmax scale has to be positive and finite, got {scale}")
    return scale


@functools.lru_cache(maxsize=1024)
def _ws_bytes(name, *sizes):
    return int(getattr(_C.load(), name)(*sizes))


def _workspace(name, device, *sizes):
    n = _ws_bytes(name, *sizes)
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    return ws, (0 if ws is None else ws.data_ptr()), n


def packed_attention(q, k, v, cu_q, cu_k, max_q: int, max_k: int, *, causal: bool = True, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None):
    """softmax(scale q k^T) v within every sequence: rows cu_q[b] .. cu_q[b + 1] of q [Tq, Hq, D] over keys cu_k[b] .. cu_k[b + 1] of
    k, v [Tk, Hkv, D] (bf16 or fp16, D 64 | 128, Hq a multiple of Hkv; query head h reads key head h // (Hq // Hkv)).  causal: row i of
    Lq sees keys j <= i + Lk - Lq; a row that sees none is 0.  scale: default D ** -0.5.

    max_q, max_k: the longest sequences' lengths or more (rows of a sequence past max_q are not computed).  out: rows that belong to
    no sequence are left as they are; without it they are 0."""
    out = _operands(q, out, k=k, v=v)
    tq, hq, dim = q.shape
    _need(k.dim() == 3 and k.shape == v.shape and k.dtype == q.dtype and v.dtype == q.dtype and k.shape[2] == dim,
          f"k, v: {q.dtype} [keys, heads, {dim}] expected, got {k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    tk, hkv, _ = k.shape
    _need(hkv > 0 and hq > 0 and hq % hkv == 0, f"{hq} query heads are no multiple of {hkv} key heads")
    batch = cu_q.shape[0] - 1 if cu_q.dim() == 1 else -1
    _need(batch >= 0, "cu_q: one entry more than there are sequences expected")
    _index("cu_q", cu_q, (batch + 1,), q.device), _index("cu_k", cu_k, (batch + 1,), q.device)
    max_q, max_k = min(int(max_q), tq), min(int(max_k), tk)
    _need(max_q >= 0 and max_k >= 0, "max_q and max_k are lengths")
    scale = _scale(scale, dim)
    if batch == 0 or max_q == 0:
        return out
    ws, ws_ptr, n = _workspace("iggt_packed_attn_ws_bytes", q.device, batch, max_q, max_k, hq, hkv, dim)
    _call("iggt_packed_attn_" + ("f16" if q.dtype == torch.float16 else "bf16"), q.device,
          q.data_ptr(), *_strides("q", q, 8), k.data_ptr(), *_strides("k", k, 8), v.data_ptr(), *_strides("v", v, 8),
          out.data_ptr(), *_strides("out", out, 4), cu_q.data_ptr(), cu_k.data_ptr(), batch, tq, tk, max_q, max_k, hq, hkv, dim,
          scale, int(causal), ws_ptr, n)
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
        _need(page in PAGE_SIZES and head_dim in HEAD_DIMS and pages >= 0 and kv_heads > 0,
              f"pages of {PAGE_SIZES} tokens and head dims {HEAD_DIMS} expected, got {page} and {head_dim}")
        make = functools.partial(torch.zeros, dtype=torch.uint8, device=device)
        return Pages(make(pages, kv_heads, page, head_dim), make(pages, kv_heads), make(pages, kv_heads, page // 16, head_dim, 16),
                     make(pages, kv_heads))


def _pages(pages, device):
    """(number of pages, key heads, page size, head dim) of a checked cache."""
    k = pages.k_codes
    _need(k.dim() == 4 and k.shape[2] in PAGE_SIZES and k.shape[3] in HEAD_DIMS,
          f"K codes: [pages, heads, {PAGE_SIZES}, {HEAD_DIMS}] expected, got {tuple(k.shape)}")
    n, heads, page, dim = k.shape
    for t, shape in ((k, k.shape), (pages.k_scale, (n, heads)), (pages.v_codes, (n, heads, page // 16, dim, 16)), (pages.v_scale, (n, heads))):
        _need(t.dtype == torch.uint8 and t.shape == shape and t.is_contiguous() and t.device == device,
              f"cache buffers: contiguous uint8 {tuple(shape)} on {device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    _need(n * page < 2 ** 31, "more than 2^31 slots")
    return n, heads, page, dim


def append_pages(pages: Pages, k, v, slots):
    """Writes k, v [T, key heads, D] (bf16 or fp16) into the cache at slots [T] (int32: page * page size + place; rows whose slot is
    not in the cache are skipped).  Rows of one page have to be one run of consecutive slots, as plan_pages gives them: a page that
    appears in two runs of one call has no defined content.  The scale of a page is the least power of two that holds its largest
    finite value, and never falls while the page is being filled; held codes are rewritten when it grows."""
    _need(k.is_cuda and k.dim() == 3 and k.dtype in _C.H16, "k: bf16 or fp16 [tokens, key heads, D] on a ROCm device expected (no CPU fallback)")
    n, heads, page, dim = _pages(pages, k.device)
    _need(v.shape == k.shape and v.dtype == k.dtype and v.device == k.device and tuple(k.shape[1:]) == (heads, dim),
          f"k, v: [tokens, {heads}, {dim}] of one type expected, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    _need(not ((k.requires_grad or v.requires_grad) and torch.is_grad_enabled()), "append_pages is forward only: an input requires gradients")
    _index("slots", slots, (k.shape[0],), k.device)
    _call("iggt_append_pages_" + ("f16" if k.dtype == torch.float16 else "bf16"), k.device,
          k.data_ptr(), *_strides("k", k, 8), v.data_ptr(), *_strides("v", v, 8), slots.data_ptr(), k.shape[0],
          pages.k_codes.data_ptr(), pages.k_scale.data_ptr(), pages.v_codes.data_ptr(), pages.v_scale.data_ptr(), n, page, heads, dim)
    return pages


def paged_attention(q, pages: Pages, tables, lens, max_q: int, max_len: int, *, cu_q=None, causal: bool = True,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None):
    """packed_attention's formula with keys and values out of the cache: request b's token t is place t % page of page
    tables[b, t // page], and it holds lens[b] of them (the new ones among them).  q [Tq, Hq, D]: rows cu_q[b] .. cu_q[b + 1] of request b
    are its last tokens; cu_q None: one row per request, row b.  causal: row i of Lq sees tokens t <= i + lens[b] - Lq.

    max_q, max_len: the largest number of rows, of tokens, or more.  Tokens on a page that does not exist count as not there.  out:
    as in packed_attention."""
    out = _operands(q, out, tables=tables, lens=lens)
    tq, hq, dim = q.shape
    n, hkv, page, d = _pages(pages, q.device)
    _need(d == dim and hq > 0 and hq % hkv == 0, f"q has {hq} heads of {dim}, the cache {hkv} of {d}")
    _need(tables.dim() == 2 and tables.dtype == _INT and (tables.shape[1] <= 1 or tables.stride(1) == 1),
          "tables: int32 [requests, pages of the longest] with contiguous rows expected")
    batch, width = tables.shape
    _index("lens", lens, (batch,), q.device)
    max_q = min(int(max_q), tq)
    if cu_q is None:
        _need(max_q <= 1 and tq >= batch, "without cu_q there is one row per request")
    else:
        _index("cu_q", cu_q, (batch + 1,), q.device)
    max_len = min(int(max_len), width * page)
    _need(max_q >= 0 and max_len >= 0 and width * page < 2 ** 31, "max_q and max_len are lengths")
    scale = _scale(scale, dim)
    if batch == 0 or max_q == 0:
        return out
    ws, ws_ptr, nbytes = _workspace("iggt_paged_attn_ws_bytes", q.device, batch, max_q, max_len, hq, hkv, dim)
    _call("iggt_paged_attn_" + ("f16" if q.dtype == torch.float16 else "bf16"), q.device,
          q.data_ptr(), *_strides("q", q, 8), out.data_ptr(), *_strides("out", out, 4),
          pages.k_codes.data_ptr(), pages.k_scale.data_ptr(), pages.v_codes.data_ptr(), pages.v_scale.data_ptr(), n, page,
          tables.data_ptr(), tables.stride(0), width, lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(), batch, tq, max_q,
          max_len, hq, hkv, dim, scale, int(causal), ws_ptr, nbytes)
    return out


def plan_pages(tables, ring, counters, lens, new_lens, page: int, tokens: int):
    """One step of the block tables: requests that hold lens [R] tokens are to hold new_lens [R] (more: tokens are appended; fewer: the
    last ones are dropped; 0: the request ends).  Growing requests take pages from the head of `ring` [N] (free pages ring[(head + i) % N],
    i < count; counters = (head, count, ...)), pages no longer needed go behind its tail for later steps, both in request order.
    tables [R, width] and ring are updated in place; lens and counters are not.

    Returns (tables, ring, starts [R + 1], next_lens [R], next_counters [3] = (head, count, missing), slots [tokens]): slots of the
    added tokens in request order, -1 behind the last, request b's at starts[b] .. starts[b + 1].  `missing` pages > 0 (or -1: `tokens` is
    too small) means that no request has grown in this step."""
    device = tables.device
    _need(tables.is_cuda, "IGGT HIP ops need tensors on a ROCm device (no CPU fallback)")
    _need(page in PAGE_SIZES, f"pages hold {PAGE_SIZES} tokens, not {page}")
    _need(tables.dim() == 2 and tables.dtype == _INT and (tables.shape[1] <= 1 or tables.stride(1) == 1) and (tables.shape[0] <= 1 or tables.stride(0) >= tables.shape[1]),
          "tables: int32 [requests, pages of the longest] with contiguous rows expected")
    requests, width = tables.shape
    tokens = int(tokens)
    _need(requests <= MAX_REQUESTS and tokens >= 0, f"at most {MAX_REQUESTS} requests")
    _need(width * page < 2 ** 31 - 128 and ring.numel() * page < 2 ** 31, "more than 2^31 slots")
    _index("ring", ring, (ring.numel(),), device)
    _need(counters.dtype == _INT and counters.device == device and counters.dim() == 1 and counters.numel() >= 2 and counters.is_contiguous(),
          "counters: int32 (head, count, ...) expected")
    _index("lens", lens, (requests,), device), _index("new_lens", new_lens, (requests,), device)
    # one allocation for the four outputs, each 16-byte aligned
    at = [0]
    for n in (requests + 1, requests, 3, tokens):
        at.append(at[-1] + (n + 3) // 4 * 4)
    buf = torch.empty(at[-1], dtype=_INT, device=device)
    starts, next_lens, next_counters, slots = (buf[a:a + n] for a, n in zip(at, (requests + 1, requests, 3, tokens)))
    base = buf.data_ptr()
    _call("iggt_plan_pages", device, tables.data_ptr(), tables.stride(0), requests, width, ring.data_ptr(), ring.numel(),
          counters.data_ptr(), lens.data_ptr(), new_lens.data_ptr(), page, base, base + 4 * at[1], base + 4 * at[2], base + 4 * at[3], tokens)
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
        _need(page in PAGE_SIZES, f"pages hold {PAGE_SIZES} tokens, not {page}")
        _need(0 < requests <= MAX_REQUESTS and longest > 0 and pages > 0, "requests, longest and pages have to be positive")
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
