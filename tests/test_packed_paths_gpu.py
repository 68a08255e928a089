"""Packed and cached attention kernel by kernel: every case first asks the host which kernel its sizes take (so that another dispatch rule
cannot move it away unseen), then compares with the 64-bit references of packed_ref.py, under the bounds derived there."""
import ctypes

import pytest
import torch

import packed_ref as R
from iggt_official_amd import _C
from iggt_official_amd.layers import Pages, append_pages, packed_attention, paged_attention
from test_packed_gpu import INF, NAN, ints, make_cache, rand

pytestmark = pytest.mark.gpu


def plan(paged, requests, rows, keys, hq, hkv, dim):
    """(rows of a work item, key ranges): 16 rows are the kernel without LDS tiles."""
    item, ranges = ctypes.c_int(), ctypes.c_int()
    assert _C.load().iggt_seq_attn_plan(int(paged), requests, rows, keys, hq, hkv, dim, item, ranges) == 0
    return item.value, ranges.value


def cached(q, pages, tables, lens, lq, causal=True, max_q=None, **kw):
    return paged_attention(q, pages, tables, ints(lens), max(lq) if max_q is None else max_q, max(lens), cu_q=R.starts(lq, "cuda"), causal=causal, **kw)


# (rows of a work item, ranges or not), dim, heads of q / of the cache, tokens held, rows
TILES = [
    (16, False, 64, 4, 2, [200, 330], [3, 3]),
    (16, False, 128, 4, 2, [200, 330], [3, 3]),
    (16, True, 64, 1, 1, [5000], [3]),
    (128, False, 64, 4, 2, [200, 330], [150, 150]),
    (128, True, 64, 1, 1, [5000], [130]),
    (256, False, 64, 16, 16, [300, 330, 500] + [16] * 37, [256, 256, 130] + [16] * 37),
    (256, True, 64, 4, 1, [5001], [1000]),
    (128, False, 128, 16, 16, [200, 330] + [40 + i for i in range(68)], [33, 40] + [i % 39 for i in range(68)]),
    (128, True, 128, 1, 1, [5000], [100]),
    (256, False, 128, 4, 2, [200, 330], [150, 150]),
    (256, True, 128, 1, 1, [5000], [200]),
]
tiles = pytest.mark.parametrize("item,split,dim,hq,hkv,lens,lq", TILES, ids=[f"{t[0]}x{t[2]}{'-ranges' if t[1] else ''}" for t in TILES])


def on_path(item, split, dim, hq, hkv, lens, lq):
    got, ranges = plan(True, len(lens), max(lq), max(lens), hq, hkv, dim)
    assert got == item and (ranges > 1) == split


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@tiles
def test_cached_attention_with_missing_pages_and_nan(item, split, dim, hq, hkv, lens, lq, causal, dt):
    """Entries outside the pool count as not there; NaN codes of held tokens reach the rows that see them and no other."""
    on_path(item, split, dim, hq, hkv, lens, lq)
    pages, tables = make_cache(lens, 32, hkv, dim, 5)
    tables[0, 1], tables[0, 4] = -1, 10 ** 6
    seen = [torch.ones(n, dtype=torch.bool, device="cuda") for n in lens]
    seen[0][32:64] = seen[0][128:160] = False
    if len(lens) > 1:
        tables[1, 0], tables[1, 10] = -7, 2 ** 30
        seen[1][:32] = seen[1][320:] = False
    last = int(tables[0, (lens[0] - 1) // 32])
    place = (lens[0] - 2) % 32
    pages.v_codes[last, 0, place // 16, 5, place % 16] = 0x7f               # the token before the last: the last two rows see it
    if hkv > 1:
        pages.k_codes[last, hkv - 1, (lens[0] - 1) % 32, 9] = 0xff          # the last token's key
    q = rand((sum(lq), hq, dim), 6, R.H16[dt])
    o = cached(q, pages, tables, lens, lq, causal)
    k, v = R.held(pages, tables, lens)
    R.close(o, *R.attention(q, k, v, lq, lens, causal, seen=seen))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 128])
@tiles
def test_cached_attention_of_every_kernel(item, split, dim, hq, hkv, lens, lq, page, dt):
    on_path(item, split, dim, hq, hkv, lens, lq)
    pages, tables = make_cache(lens, page, hkv, dim, 9)
    q = rand((sum(lq), hq, dim), 10, R.H16[dt], 1.5)
    k, v = R.held(pages, tables, lens)
    for causal in (True, False):
        R.close(cached(q, pages, tables, lens, lq, causal), *R.attention(q, k, v, lq, lens, causal))


@pytest.mark.parametrize("item,dim,held,rows", [(128, 64, 230, 250), (256, 128, 230, 200), (128, 128, 4200, 100)])
def test_cached_tiles_beyond_4_gib(item, dim, held, rows):
    """A pool of more than 4 GB of codes: the pages in use lie at its two ends and in its middle."""
    heads, page = 16, 64
    total = 70000 * 64 // dim
    assert plan(True, 1, rows, held, heads, heads, dim)[0] == item
    pages = Pages.empty(total, heads, dim, page)
    assert pages.k_codes.numel() > 2 ** 32
    ids = [(total - 1 - i // 3, i // 3, total // 2 + i // 3)[i % 3] for i in range(-(-held // page))]
    kv = rand((held, 2, heads, dim), 1, torch.float16)
    append_pages(pages, kv[:, 0], kv[:, 1], ints([ids[i // page] * page + i % page for i in range(held)]))
    q = rand((rows, heads, dim), 2, torch.float16)
    o = cached(q, pages, ints([ids]), [held], [rows])
    few = Pages(*(t[ids].contiguous() for t in pages))
    k, v = R.held(few, ints([list(range(len(ids)))]), [held])
    R.close(o, *R.attention(q, k, v, [rows], [held], True))


@pytest.mark.parametrize("item,dim,heads,rows", [(16, 64, 1, 20), (128, 64, 1, 200), (256, 64, 512, 130), (256, 128, 1, 200)])
@pytest.mark.parametrize("dt,sizes", [("f16", (65504.0, 1.0, 3e-5)), ("bf16", (1e30, 1.0, 1e-30))])
def test_cached_tiles_of_v_at_the_edges_of_the_types(item, dim, heads, rows, dt, sizes):
    """fp16: V up to 65 504 (its e4m3 neighbour is 65 536) and down to the subnormals; bf16: 1e30 and 1e-30 in one cache."""
    pages = Pages.empty(3, heads, dim, 64)
    k, v = rand((192, heads, dim), 1, R.H16[dt]), rand((192, heads, dim), 2, torch.float32).clamp(-1, 1)
    v = (v * torch.tensor(sizes, device="cuda").repeat_interleave(64)[:, None, None]).to(R.H16[dt])
    append_pages(pages, k, v, torch.arange(192, dtype=torch.int32, device="cuda"))
    q = rand((rows, heads, dim), 3, R.H16[dt])
    for n in (64, 128, 192):                         # (the last keys alone decide where large values would hide the small ones)
        assert plan(True, 1, rows, n, heads, heads, dim)[0] == item
        tables = ints([[2, 1, 0][:n // 64]])
        kk, vv = R.held(pages, tables, [n])
        R.close(cached(q, pages, tables, [n], [rows], False), *R.attention(q, kk, vv, [rows], [n], False))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("paged,item,split,dim,heads,n,lq", [
    (False, 128, True, 64, 1, 5001, 1), (False, 128, True, 128, 1, 5001, 70), (False, 128, False, 64, 70, 700, 190), (False, 128, False, 128, 70, 700, 190),
    (False, 256, False, 64, 300, 400, 300), (True, 16, True, 64, 1, 5001, 1), (True, 16, True, 128, 2, 5001, 7), (True, 16, True, 64, 1, 60001, 1),
    (True, 128, True, 64, 1, 5001, 130), (True, 256, True, 64, 4, 5001, 1000), (True, 128, True, 128, 1, 5001, 100), (True, 256, True, 128, 1, 5001, 200)])
def test_every_key_at_a_tiles_end_counts_once(paged, item, split, dim, heads, n, lq, causal, dt):
    """The first and the last key of every 64 (and so of every key range) hold all the weight, each with a channel of V of its own (or one
    of a few that share one): a key that is dropped or read twice moves its channel by a tenth or more."""
    got, ranges = plan(paged, 1, lq, n, heads, heads, dim)
    assert got == item and (ranges > 1) == split
    dtype = R.H16[dt]
    at = torch.arange(n, device="cuda")
    ends = ((at % 64 == 0) | (at % 64 == 63) | (at == n - 1)) & ((at // 64 % -(-n // 5001)) == 0)
    place = torch.cumsum(ends, 0) - 1
    k, v = torch.zeros(n, heads, dim, dtype=dtype, device="cuda"), torch.zeros(n, heads, dim, dtype=dtype, device="cuda")
    k[ends] = 4.0
    v[at[ends], :, place[ends] % dim] = 1.0
    q = torch.full((lq, heads, dim), 40.0 / dim ** 0.5 / 8, dtype=dtype, device="cuda")      # scores 20 above the others'
    if paged:
        pages = Pages.empty(-(-n // 64), heads, dim, 64)
        append_pages(pages, k, v, at.int())
        o = cached(q, pages, torch.arange(-(-n // 64), dtype=torch.int32, device="cuda")[None], [n], [lq], causal)
    else:
        o = packed_attention(q, k, v, R.starts([lq], "cuda"), R.starts([n], "cuda"), lq, n, causal=causal)
    ref, tol = R.attention(q, k, v, [lq], [n], causal)
    assert float(tol.max()) < 0.02 * float(ref.max())
    R.close(o, ref, tol)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,heads,lens", [(64, 2, [100, 300, 64]), (64, 80, [100, 300, 64]), (64, 640, [100, 7]), (64, 640, [128, 500]), (128, 2, [100, 300, 64]), (128, 640, [100, 7])])
def test_packed_tiles_of_128_rows_on_small_and_full_grids(dim, heads, lens, causal, dt):
    """64 channels: up to two waves per SIMD are pipelined over the tiles, more are not.  NaN among the values that only later rows see."""
    lk = [n + 70 for n in lens]
    if heads == 640:
        lens = [min(n, 128) for n in lens]
    assert plan(False, len(lens), max(lens), max(lk), heads, heads, dim) == (128, 1)
    q, k, v = rand((sum(lens), heads, dim), 1, R.H16[dt], 1.5), rand((sum(lk), heads, dim), 2, R.H16[dt]), rand((sum(lk), heads, dim), 3, R.H16[dt])
    v[lk[0] - 2, 0, 5], v[lk[0] - 1, heads - 1, 9], k[lk[0] - 1, 1, 2] = NAN, -INF, NAN
    o = packed_attention(q, k, v, R.starts(lens, "cuda"), R.starts(lk, "cuda"), max(lens), max(lk), causal=causal)
    R.close(o, *R.attention(q, k, v, lens, lk, causal))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("page,heads,dim,tokens", [(64, 16, 64, 9000), (16, 17, 128, 9000), (128, 2, 64, 70000)])
def test_append_pages_of_a_prompt_in_groups_of_64(page, heads, dim, tokens, dt):
    """As many tokens and heads as make a workgroup look at 64 slots: whole pages in any order, rows that go nowhere in front."""
    total = -(-tokens // page)
    assert tokens // 64 * ((heads + 1) // 2) >= 1024
    order = torch.randperm(total, generator=torch.Generator().manual_seed(1)).cuda()
    t = torch.arange(tokens, device="cuda")
    slots = (order[t // page] * page + t % page).int()
    pages = Pages.empty(total, heads, dim, page)
    kv = rand((tokens + 37, 2, heads, dim), 2, R.H16[dt], 3.0)
    append_pages(pages, kv[:, 0], kv[:, 1], torch.cat([torch.full((37,), -1, dtype=torch.int32, device="cuda"), slots]))
    k, v = (x.cuda() for x in R.code_values(pages))
    for codes, byte, x in ((k, pages.k_scale, kv[37:, 0]), (v, pages.v_scale, kv[37:, 1])):
        whole = torch.zeros(total * page, heads, dim, dtype=torch.float64, device="cuda")
        whole[slots.long()] = x.double()
        whole = whole.view(total, page, heads, dim).transpose(1, 2)
        m, e = torch.frexp(whole.abs().amax((2, 3)))                     # 448 = 0.875 * 2^9
        need = torch.where(m > 0, e - 9 + (m > 0.875).int() + 127, 1).clamp(1, 254)
        assert torch.equal(byte.int(), need.int())
        assert torch.equal(codes, R.e4m3(whole * torch.exp2(127.0 - need.double())[..., None, None]))
