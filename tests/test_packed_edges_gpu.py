"""Packed and cached attention at the borders of what their documentation allows, against the 64-bit references of packed_ref.py."""
import pytest
import torch

import packed_ref as R
from iggt_official_amd.layers import Pages, append_pages, packed_attention, paged_attention, plan_pages
from test_packed_gpu import INF, NAN, ints, make_cache, rand
from test_packed_paths_gpu import cached, plan

pytestmark = pytest.mark.gpu


def first_rows(lq, max_q):
    """Mask over the packed rows: the first max_q of every sequence."""
    return torch.cat([torch.arange(n) < max_q for n in lq]).cuda()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,hq,hkv,lq,lk,max_q,item", [
    (64, 2, 2, [64], [64], 10, 128), (128, 4, 1, [64, 5, 30], [64, 40, 12], 10, 128), (64, 16, 16, [400] * 40, [400] * 40, 270, 256),
    (64, 1, 1, [900], [5000], 130, 128), (128, 2, 2, [3], [6000], 1, 128)])
def test_packed_rows_behind_max_q_do_not_move_the_mask(dim, hq, hkv, lq, lk, max_q, item, dt):
    """Of a sequence longer than max_q the first rows are computed, under the mask of the whole sequence; the others stay as they are."""
    assert plan(False, len(lq), max_q, max(lk), hq, hkv, dim)[0] == item
    q, k, v = rand((sum(lq), hq, dim), 1, R.H16[dt]), rand((sum(lk), hkv, dim), 2, R.H16[dt]), rand((sum(lk), hkv, dim), 3, R.H16[dt])
    v[lk[0] - 1] = NAN                               # only the last row of the first sequence sees it
    few = first_rows(lq, max_q)
    out = torch.full_like(q, 3.0)
    packed_attention(q, k, v, R.starts(lq, "cuda"), R.starts(lk, "cuda"), max_q, max(lk), out=out)
    ref, tol = R.attention(q, k, v, lq, lk, True)
    R.close(out[few], ref[few], tol[few])
    assert (out[~few] == 3).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,hq,hkv,lq,lens,max_q,item", [
    (64, 4, 2, [3, 9, 1, 0], [70, 200, 20, 9], 1, 16), (128, 4, 4, [30, 9], [300, 200], 2, 16), (64, 2, 1, [64], [64], 10, 16), (128, 1, 1, [40], [6000], 1, 16),
    (64, 4, 2, [200, 300], [250, 300], 150, 128), (64, 32, 32, [150] * 16, [200] * 16, 130, 256), (128, 4, 2, [200, 300], [250, 300], 150, 256),
    (128, 1, 1, [150], [5000], 100, 128)])
def test_cached_rows_behind_max_q_do_not_move_the_mask(dim, hq, hkv, lq, lens, max_q, item, dt):
    assert plan(True, len(lq), max_q, max(lens), hq, hkv, dim)[0] == item
    pages, tables = make_cache(lens, 16, hkv, dim, 4)
    last = lens[0] - 1                               # a NaN that only the last row of the first request sees
    pages.v_codes[int(tables[0, last // 16]), 0, 0, 7, last % 16] = 0x7f
    q = rand((sum(lq), hq, dim), 5, R.H16[dt])
    few = first_rows(lq, max_q)
    out = torch.full_like(q, 3.0)
    cached(q, pages, tables, lens, lq, max_q=max_q, out=out)
    k, v = R.held(pages, tables, lens)
    ref, tol = R.attention(q, k, v, lq, lens, True)
    R.close(out[few], ref[few], tol[few])
    assert (out[~few] == 3).all()


KERNELS = pytest.mark.parametrize("item,dim,heads,rows", [(16, 64, 1, 20), (16, 128, 1, 1), (128, 64, 1, 200), (256, 64, 512, 130), (256, 128, 1, 200), (128, 128, 16, 100)])


@pytest.mark.parametrize("size,of_q,scale", [(1e6, 1e-5, None), (1e-6, 3e4, 4.0), (3e-8, 3e4, 120.0)])
@KERNELS
def test_fp16_rows_over_keys_beyond_the_range_of_fp16(item, dim, heads, rows, size, of_q, scale):
    """A cache written from bf16 holds keys that fp16 does not: their scores are formed from the codes, the scale goes on in fp32."""
    n = 4200 if (item, dim) == (128, 128) else 190
    assert plan(True, 1, rows, n, heads, heads, dim)[0] == item
    g = torch.Generator(device="cuda").manual_seed(3)
    k = (torch.randn(n, heads, dim, device="cuda", generator=g) * size).bfloat16()
    k[16:32] *= 0.25                                 # (pages of other scales beside them)
    v = rand((n, heads, dim), 4, torch.bfloat16)
    pages = Pages.empty(-(-n // 16), heads, dim, 16)
    append_pages(pages, k, v, torch.arange(n, dtype=torch.int32, device="cuda"))
    tables = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None]
    q = (torch.randn(rows, heads, dim, device="cuda", generator=g).clamp(-2, 2) * of_q).half()
    kk, vv = R.held(pages, tables, [n])
    for causal in (True, False):
        R.close(cached(q, pages, tables, [n], [rows], causal, scale=scale), *R.attention(q, kk, vv, [rows], [n], causal, scale=scale))


@pytest.mark.parametrize("paged,rows,lk", [(True, 1, 2000), (True, 1, 20000), (True, 5, 2000), (True, 5, 20000), (True, 200, 20000), (False, 1, 2000), (False, 1, 20000)])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_in_a_key_range_whose_weight_vanishes(paged, rows, lk, dim, dt):
    """One key outweighs all others by 2^250: a NaN among those still reaches the rows that see it, whatever number of key ranges there is."""
    q, k, v = rand((rows, 1, dim), 1, R.H16[dt], 0.1), rand((lk, 1, dim), 2, R.H16[dt], 0.1), rand((lk, 1, dim), 3, R.H16[dt])
    q[:, :, 0], k[:, :, 0] = 16.0, 0.0
    k[5, 0, 0] = 192.0 / 16 * dim ** 0.5
    v[lk // 2 + 9, 0, 11] = NAN
    if paged:
        pages = Pages.empty(-(-lk // 64), 1, dim, 64)
        append_pages(pages, k, v, torch.arange(lk, dtype=torch.int32, device="cuda"))
        tables = torch.arange(-(-lk // 64), dtype=torch.int32, device="cuda")[None]
        o = cached(q, pages, tables, [lk], [rows])
        k, v = R.held(pages, tables, [lk])
    else:
        o = packed_attention(q, k, v, R.starts([rows], "cuda"), R.starts([lk], "cuda"), rows, lk)
    assert (plan(paged, 1, rows, lk, 1, 1, dim)[1] > 8) == (lk == 20000)
    R.close(o, *R.attention(q, k, v, [rows], [lk], True))


@pytest.mark.parametrize("item,dim,heads,rows", [(16, 64, 2, 3), (16, 128, 1, 20), (128, 64, 1, 200), (256, 64, 512, 130), (256, 128, 1, 200)])
def test_fp16_rows_over_values_beyond_the_range_of_fp16(item, dim, heads, rows):
    """V beyond 131 008 is infinite for fp16 rows: for those that see it."""
    n = 190
    assert plan(True, 1, rows, n, heads, heads, dim)[0] == item
    k, v = rand((n, heads, dim), 1, torch.bfloat16), rand((n, heads, dim), 2, torch.bfloat16)
    v[n - 1, 0, 3], v[n - 1, 0, 4], v[n - 2, 0, 5], v[n - 2, 0, 6], v[n - 1, 0, 6], v[n - 2, 0, 7] = 4e5, -4e5, 3e5, 3e5, -3e5, NAN
    pages = Pages.empty(12, heads, dim, 16)
    append_pages(pages, k, v, torch.arange(n, dtype=torch.int32, device="cuda"))
    tables = torch.arange(12, dtype=torch.int32, device="cuda")[None]
    q = rand((rows, heads, dim), 3, torch.float16)
    kk, vv = R.held(pages, tables, [n])
    vv = torch.where(vv.abs() > 131008, vv.sign() * INF, vv)
    for causal in (True, False):
        R.close(cached(q, pages, tables, [n], [rows], causal), *R.attention(q, kk, vv, [rows], [n], causal))


@pytest.mark.parametrize("dim", [64, 128])
def test_one_key_has_no_row_stride(dim):
    """One row of a very wide matrix as K and V: the distance to a row that is not there does not matter."""
    wide = torch.zeros(2 ** 24 + 4 * dim, dtype=torch.float16, device="cuda")
    kv = wide.as_strided((1, 2, dim), (2 ** 24, dim, 1))
    kv.copy_(rand((1, 2, dim), 1, torch.float16))
    q = rand((3, 2, dim), 2, torch.float16)
    o = packed_attention(q, kv, kv, R.starts([3], "cuda"), R.starts([1], "cuda"), 3, 1, causal=False)
    R.close(o, *R.attention(q, kv, kv, [3], [1], False))


def test_packed_grid_of_more_than_32_bits_of_threads():
    """One long prompt among 70 000 sequences of one token: 16 x 70 001 x 8 work items of 512 threads."""
    n, heads, long = 70000, 8, 4000
    lens = [1] * (n // 2) + [long] + [1] * (n // 2)
    assert plan(False, n + 1, long, long, heads, heads, 64) == (256, 1)
    q, k, v = (rand((n + long, heads, 64), i, torch.float16) for i in range(3))
    cu = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(torch.tensor(lens), 0)]).int().cuda()
    o = packed_attention(q, k, v, cu, cu, long, long)
    s = slice(n // 2, n // 2 + long)
    R.close(o[s], *R.attention(q[s], k[s], v[s], [long], [long], True))
    assert torch.equal(o[:n // 2], v[:n // 2]) and torch.equal(o[n // 2 + long:], v[n // 2 + long:])


def test_cached_grid_of_more_than_32_bits_of_threads():
    """A row for each of 2^20 + 1 requests of 16 heads, 256 threads each; all of them hold the same token."""
    n, heads = 2 ** 20 + 1, 16
    assert plan(True, n, 1, 1, heads, heads, 64) == (16, 1)
    pages = Pages.empty(1, heads, 64, 16)
    k, v = rand((1, heads, 64), 1, torch.float16), rand((1, heads, 64), 2, torch.float16)
    append_pages(pages, k, v, ints([0]))
    _, value = R.held(pages, ints([[0]]), [1])
    q = torch.zeros(n, heads, 64, dtype=torch.float16, device="cuda")
    o = paged_attention(q, pages, torch.zeros(n, 1, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda"), 1, 1)
    assert (o == value.half()).all()


def test_planner_of_many_requests_in_a_captured_graph():
    """More requests than the default of dynamic LDS holds: captured, and replayed with eager work in between, it plans what an eager call does."""
    n, page, width = 5000, 16, 3
    new = ints([(7 * i) % 49 for i in range(n)])
    state = [torch.full((n, width), -1, dtype=torch.int32, device="cuda"), torch.randperm(3 * n).int().cuda(), ints([0, 3 * n]), ints([0] * n)]
    first = [t.clone() for t in state]
    want = [t.clone() for t in plan_pages(*state, new, page, 49 * n)]
    for t, old in zip(state, first):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = plan_pages(*state, new, page, 49 * n)
    for _ in range(3):
        for t, old in zip(state, first):
            t.copy_(old)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
