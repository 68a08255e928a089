"""Packed-sequence attention, the page planner, the cache writer and cached attention on the GPU, against 64-bit references on the
same operands (packed_ref.py, where the bounds are derived)."""
import pytest
import torch

import packed_ref as R
from iggt_official_amd import _C
from iggt_official_amd.layers import PagedKVCache, Pages, append_pages, packed_attention, paged_attention, plan_pages

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def rand(shape, seed, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def run_packed(lq, lk, hq, hkv, dim, dt, causal, seed=0, scale=None):
    dtype = R.H16[dt]
    q = rand((sum(lq), hq, dim), seed, dtype, 1.5)
    kv = rand((max(1, sum(lk)), 2, hkv, dim), seed + 1, dtype)
    k, v = kv[:, 0], kv[:, 1]
    o = packed_attention(q, k, v, R.starts(lq, "cuda"), R.starts(lk, "cuda"), max(lq), max(lk), causal=causal, scale=scale)
    R.close(o, *R.attention(q, k, v, lq, lk, causal, scale))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 16, 16), (64, 6, 2), (128, 4, 4), (128, 8, 1), (64, 1, 1), (128, 5, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([0, 3, 1, 0, 65], [0, 3, 64, 5, 0]), ([130, 31, 257], [130, 96, 200]), ([5, 64, 33], [2, 640, 31])])
def test_packed_attention(dt, dim, hq, hkv, causal, lq, lk):
    """Lengths of none, one, a tile, one more; more keys than rows and fewer (rows that see none)."""
    run_packed(lq, lk, hq, hkv, dim, dt, causal)


@pytest.mark.parametrize("dt,dim,hq,hkv,lq,lk", [
    ("bf16", 64, 16, 16, [300] * 32, [300] * 32), ("f16", 64, 16, 16, [277] * 40 + [1], [277] * 40 + [400]),    # 256-row tiles
    ("f16", 128, 8, 2, [1374], [1374]), ("bf16", 64, 32, 8, [700, 91], [1400, 91]),
    ("bf16", 128, 2, 2, [1], [9001]), ("f16", 64, 4, 1, [3], [20000]), ("bf16", 64, 1, 1, [200], [5000])])      # key ranges
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_larger_grids(dt, dim, hq, hkv, lq, lk, causal):
    run_packed(lq, lk, hq, hkv, dim, dt, causal, seed=5)


@pytest.mark.parametrize("scale", [1e-3, 4.0])
def test_packed_attention_scale(scale):
    """A flat and a one-hot softmax (the running maximum moves by far more than the rescale threshold)."""
    run_packed([100, 300], [100, 333], 2, 1, 64, "f16", True, seed=9, scale=scale)


def test_packed_attention_strides_and_rows_outside():
    """Operands inside a fused qkv matrix; output inside a wider one; rows before the first and behind the last sequence keep their
    content, and an output that is not given is 0 there."""
    qkv = rand((200, 3, 4, 64), 3, torch.float16)
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    cu = torch.tensor([7, 50, 50, 180], dtype=torch.int32, device="cuda")
    wide = torch.full((200, 4, 128), 7.0, dtype=torch.float16, device="cuda")
    out = wide[:, :, 64:]
    assert packed_attention(q, k, v, cu, cu, 130, 130, out=out) is out
    ref, tol = R.attention(q[7:180], k[7:180], v[7:180], [43, 0, 130], [43, 0, 130], True)
    R.close(out[7:180], ref, tol)
    assert (wide[:, :, :64] == 7).all() and (out[:7] == 7).all() and (out[180:] == 7).all()
    fresh = packed_attention(q, k, v, cu, cu, 130, 130)
    assert torch.equal(fresh[7:180], out[7:180]) and (fresh[:7] == 0).all() and (fresh[180:] == 0).all()


def test_packed_attention_one_head_with_odd_strides():
    """Dimensions of one entry have no stride: a [T, 1, D] view whose head stride is no multiple of 8."""
    base = rand((50, 64), 4, torch.bfloat16)
    q = base.as_strided((50, 1, 64), (64, 3, 1))
    cu = R.starts([50], "cuda")
    o = packed_attention(q, q, q, cu, cu, 50, 50)
    R.close(o, *R.attention(q, q, q, [50], [50], True))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,rep", [(64, 1), (128, 1), (64, 40)])
def test_packed_attention_not_finite(dt, dim, rep):
    """inf and NaN in K and V reach the rows that see them and no other: keys of other sequences, later keys, keys behind the end.
    rep 40: the 256-row tiles."""
    lens = [70, 150, 260] if rep == 1 else [300] * rep
    hq = hkv = 2 if rep == 1 else 16
    q, k, v = (rand((sum(lens), hq, dim), 11 + i, R.H16[dt]) for i in range(3))
    v[40, 0, 3], v[41, 0, 3], v[60, 1, 5], v[200, 0, 63], v[sum(lens) - 1, 1, 0] = INF, -INF, NAN, -INF, INF
    v[sum(lens) - 2] = NAN
    k[65, 0, 1], k[210, 1, 2] = NAN, NAN
    for causal in (True, False):
        o = packed_attention(q, k, v, R.starts(lens, "cuda"), R.starts(lens, "cuda"), max(lens), max(lens), causal=causal)
        few = lens if rep == 1 else lens[:2]
        n = sum(few)
        ref, tol = R.attention(q[:n], k[:n], v[:n], few, few, causal)
        R.close(o[:n], ref, tol)
        if rep > 1:
            last = slice(sum(lens) - 300, None)
            R.close(o[last], *R.attention(q[last], k[last], v[last], [300], [300], causal))
            assert o[n:sum(lens) - 300].isfinite().all()


def test_packed_attention_ignores_what_no_sequence_holds():
    """Prefix sums are clamped to the tensors; rows behind max_q are not computed."""
    q, k, v = (rand((64, 2, 64), 20 + i, torch.float16) for i in range(3))
    bad = torch.tensor([-5, 30, 20, 1000], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    packed_attention(q, k, v, bad, bad, 64, 64, out=out)
    R.close(out[:20], *[x[:20] for x in R.attention(q[:30], k[:30], v[:30], [30], [30], True)])
    # (rows 20 .. 29 belong to two of these sequences: either's)
    R.close(out[30:], *[x[10:] for x in R.attention(q[20:], k[20:], v[20:], [44], [44], True)])
    out.fill_(3.0)
    packed_attention(q, k, v, R.starts([64], "cuda"), R.starts([64], "cuda"), 10, 64, out=out)
    assert (out[10:] == 3).all()


def test_packed_attention_refusals():
    q, cu = rand((8, 4, 64), 1, torch.float16), R.starts([8], "cuda")
    ok = lambda **kw: packed_attention(**{**dict(q=q, k=q, v=q, cu_q=cu, cu_k=cu, max_q=8, max_k=8), **kw})  # noqa: E731
    ok()
    for kw in (dict(q=q.float()), dict(k=q.bfloat16()), dict(v=q[:4]), dict(k=q[:, :3], v=q[:, :3]), dict(q=q[..., :32], k=q[..., :32], v=q[..., :32]),
               dict(cu_q=cu.long()), dict(cu_k=R.starts([4, 4], "cuda")), dict(cu_q=cu.cpu()), dict(scale=0.0), dict(scale=NAN), dict(max_q=-1),
               dict(out=torch.empty_like(q[:4])), dict(out=q.float()), dict(out=q[:1].expand(8, 4, 64)),
               dict(q=rand((8, 4, 66), 1, torch.float16)[..., :64]), dict(q=rand((8, 4 * 64 + 4), 1, torch.float16)[:, 4:].view(8, 4, 64)),
               dict(q=q.clone().requires_grad_())):
        with pytest.raises(_C.HipExtensionError):
            ok(**kw)
    with torch.no_grad():
        ok(q=q.clone().requires_grad_())
    empty = q[:0]
    assert packed_attention(empty, q, q, R.starts([0], "cuda"), cu, 0, 8).shape == (0, 4, 64)
    assert (packed_attention(q, q, q, cu[:1], cu[:1], 8, 8) == 0).all()
    assert (ok(k=empty, v=empty, cu_k=R.starts([0], "cuda"), max_k=0) == 0).all()


# ------------------------------------------------------------------------------------------------ cache
def make_cache(lens, page, heads, dim, seed=0, spare=3, fill=0x7f):
    """Shuffled pages whose places behind the ends hold `fill` (NaN codes)."""
    g = torch.Generator().manual_seed(seed)
    count = [-(-n // page) for n in lens]
    total = sum(count) + spare
    perm = torch.randperm(total, generator=g).int()
    width = max(max(count), 1) + 1
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        tables[b, :c] = perm[at:at + c]
        at += c
    scale = [torch.randint(119, 124, (total, heads), generator=g).to(torch.uint8) for _ in range(2)]
    value = [torch.randn(total, heads, page, dim, generator=g) * torch.exp2(127.0 - s.float())[..., None, None] for s in scale]
    code = [x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for x in value]
    live = torch.zeros(total, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(count[b]):
            live[tables[b, j], :min(page, n - j * page)] = True
    code = [torch.where(live[:, None, :, None], c, fill) for c in code]
    v = code[1].view(total, heads, page // 16, 16, dim).permute(0, 1, 2, 4, 3).contiguous()
    return Pages(code[0].cuda(), scale[0].cuda(), v.cuda(), scale[1].cuda()), tables.cuda()


def run_paged(lens, lq, page, hq, hkv, dim, dt, causal, seed=0):
    pages, tables = make_cache(lens, page, hkv, dim, seed)
    q = rand((sum(lq), hq, dim), seed + 1, R.H16[dt], 1.5)
    one = all(n == 1 for n in lq)
    o = paged_attention(q, pages, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lq), max(lens),
                        cu_q=None if one and seed % 2 else R.starts(lq, "cuda"), causal=causal)
    k, v = R.held(pages, tables, lens)
    R.close(o, *R.attention(q, k, v, lq, lens, causal))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 16, 16), (64, 8, 2), (128, 4, 4), (128, 16, 1), (64, 5, 1)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [0, 15, 16, 17], [63, 64, 65, 0, 700], [3000, 1]])
def test_paged_attention_single_tokens(dt, dim, hq, hkv, page, lens):
    """One row per request: lengths of none, one, around a group of 16 and a block of 64, and split over key ranges."""
    run_paged(lens, [1] * len(lens), page, hq, hkv, dim, dt, True, seed=len(lens))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 4, 4), (128, 4, 1), (64, 24, 2)])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,lq", [([5, 70, 0, 33], [3, 4, 0, 2]), ([200, 90, 700], [150, 90, 1]), ([40, 2], [40, 6]), ([2500, 31], [300, 31])])
def test_paged_attention_many_rows(dt, dim, hq, hkv, page, causal, lens, lq):
    """Few rows (drafts) and many (a view that joins); a whole prompt; more rows than tokens (the first see none)."""
    run_paged(lens, lq, page, hq, hkv, dim, dt, causal, seed=3)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_paged_attention_256_row_tiles(dt):
    run_paged([400 + i for i in range(40)], [290] * 40, 64, 16, 16, 64, dt, True, seed=8)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_attention_bad_pages_and_nan(dt, rows, dim):
    """Entries outside the pool: their tokens count as not there.  NaN codes of held tokens reach the rows that see them only."""
    lens, page = [200, 330], 32
    pages, tables = make_cache(lens, page, 2, dim, 5)
    tables[0, 1], tables[1, 4], tables[1, 0], tables[1, 10] = -1, 10 ** 6, -7, 2 ** 30
    last = int(tables[0, 6])
    pages.v_codes[last, 0, 0, 5, 6] = 0x7f                   # token 198 of request 0: seen by the last two rows
    pages.k_codes[last, 1, 7, 9] = 0xff                      # token 199
    q = rand((2 * rows, 4, dim), 6, R.H16[dt])
    o = paged_attention(q, pages, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), rows, 330, cu_q=R.starts([rows, rows], "cuda"))
    seen = [torch.ones(n, dtype=torch.bool, device="cuda") for n in lens]
    seen[0][32:64] = False
    seen[1][:32] = seen[1][128:160] = seen[1][320:] = False
    k, v = R.held(pages, tables, lens)
    ref, tol = R.attention(q, k, v, [rows, rows], lens, True, seen=seen)
    R.close(o, ref, tol)


def test_paged_attention_only_bad_pages_and_long_lengths():
    """No page at all: 0.  Lengths beyond the table are cut to it, negative ones are none."""
    pages, tables = make_cache([100, 100], 16, 1, 64, 2)
    q = rand((2, 1, 64), 7, torch.float16)
    o = paged_attention(q, pages, torch.full_like(tables, -1), torch.tensor([100, 100], dtype=torch.int32, device="cuda"), 1, 100)
    assert (o == 0).all()
    o = paged_attention(q, pages, tables, torch.tensor([2 ** 31 - 1, -4], dtype=torch.int32, device="cuda"), 1, 2 ** 31 - 1)
    k, v = R.held(pages, tables, [112, 0])
    seen = [torch.arange(112, device="cuda") < 112, torch.ones(0, dtype=torch.bool, device="cuda")]
    assert (o[1] == 0).all()
    assert o[0].isnan().any() == R.attention(q, k, v, [1, 1], [112, 0], True, seen=seen)[0][0].isnan().any()


def test_paged_attention_refusals():
    pages, tables = make_cache([40, 40], 16, 2, 64)
    lens = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    q = rand((2, 4, 64), 1, torch.float16)
    ok = lambda **kw: paged_attention(**{**dict(q=q, pages=pages, tables=tables, lens=lens, max_q=1, max_len=40), **kw})  # noqa: E731
    ok()
    wrong = rand((2, 4, 128), 1, torch.float16)
    for kw in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=wrong), dict(tables=tables.long()), dict(tables=tables[0]), dict(lens=lens[:1]), dict(max_q=2),
               dict(q=q[:1]), dict(cu_q=R.starts([1], "cuda"), max_q=1), dict(scale=-1.0), dict(lens=lens.cpu()), dict(max_len=-1),
               dict(pages=pages._replace(v_codes=pages.v_codes[:-1])), dict(pages=pages._replace(k_scale=pages.k_scale.int())),
               dict(pages=pages._replace(k_codes=pages.k_codes[:, :, :8])), dict(q=q.clone().requires_grad_())):
        with pytest.raises(_C.HipExtensionError):
            ok(**kw)


def check_codes(pages, ref):
    k, v = R.code_values(pages)
    for got, want in ((k, ref.code[0]), (v, ref.code[1])):
        assert torch.equal(got.nan_to_num(1e9), want.nan_to_num(1e9))
    assert torch.equal(pages.k_scale.cpu().long(), ref.byte[0]) and torch.equal(pages.v_scale.cpu().long(), ref.byte[1])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,dim", [(3, 64), (2, 128), (1, 64)])
def test_append_pages_is_the_definition(dt, page, heads, dim):
    """Codes and exponents bit for bit, over calls that begin pages, fill them one token at a time with growing and falling values,
    cross them, skip slots, and hold infinities, NaN, zeros and the smallest values."""
    total = 9
    pages, ref = Pages.empty(total, heads, dim, page), R.CacheRef(total, heads, page, dim)
    order = [4, 0, 7, 2, 8, 1]                   # pages of one request, in order
    slot = lambda i: order[i // page] * page + i % page  # noqa: E731
    at = 0
    for step, (n, size) in enumerate([(1, 1.0), (3, 1e-3), (1, 50.0), (page, 4.0), (2 * page + 5, 2.0), (1, 1e4), (16, 1e4), (7, 0.0), (1, 1e-30)]):
        k, v = rand((n + 2, heads, dim), 100 + step, R.H16[dt], size), rand((n + 2, heads, dim), 200 + step, R.H16[dt], size)
        if step == 4:
            k[1, 0, 3], k[2, 0, 4], v[3, 0, 5], v[0, 0, 6] = INF, -INF, NAN, INF
        slots = [slot(at + i) for i in range(n)]
        slots = [-1] + slots + [total * page]    # rows that go nowhere
        append_pages(pages, k, v, torch.tensor(slots, dtype=torch.int32, device="cuda"))
        ref.append(k, v, slots)
        at += n
        check_codes(pages, ref)


@pytest.mark.parametrize("tokens", [40, 9000])
def test_append_pages_of_many_requests(tokens):
    """Single tokens of many pages in one call, and a long prompt beside them (both launch forms), operands in a fused matrix."""
    page, heads, dim = 16, 4, 64
    total = 64 + -(-tokens // page)
    pages, ref = Pages.empty(total, heads, dim, page), R.CacheRef(total, heads, page, dim)
    slots = [p * page for p in range(0, 64, 3)] + [64 * page + i for i in range(tokens)] + [p * page for p in range(1, 64, 3)]
    kv = rand((len(slots), 2, heads, dim), 3, torch.bfloat16, 3.0)
    append_pages(pages, kv[:, 0], kv[:, 1], torch.tensor(slots, dtype=torch.int32, device="cuda"))
    ref.append(kv[:, 0], kv[:, 1], slots)
    check_codes(pages, ref)


def test_append_pages_rounding_bound():
    """A value within a page's range is off by half an e4m3 step (2^-4 relative), or half the smallest step of the scale (2^-10)."""
    pages = Pages.empty(4, 1, 64, 64)
    k, v = rand((256, 1, 64), 1, torch.float16, 3.0), rand((256, 1, 64), 2, torch.float16, 0.01)
    append_pages(pages, k, v, torch.arange(256, dtype=torch.int32, device="cuda"))
    tables = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    for got, x, byte in zip(R.held(pages, tables, [256]), (k, v), (pages.k_scale, pages.v_scale)):
        step = torch.exp2(byte.double() - 127).view(4, 1).repeat_interleave(64, 0)[..., None]
        assert ((got - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)).all()


def test_append_pages_refusals():
    pages = Pages.empty(2, 2, 64, 16)
    k, slots = rand((4, 2, 64), 1, torch.float16), torch.arange(4, dtype=torch.int32, device="cuda")
    append_pages(pages, k, k, slots)
    append_pages(pages, k[:0], k[:0], slots[:0])
    for args in ((pages, k.float(), k.float(), slots), (pages, k, k[:2], slots), (pages, k, k, slots.long()), (pages, k, k, slots[:2]),
                 (pages, k[:, :1], k[:, :1], slots), (pages, k, k.bfloat16(), slots), (pages._replace(v_scale=pages.v_scale[:1]), k, k, slots),
                 (pages, k.clone().requires_grad_(), k, slots)):
        with pytest.raises(_C.HipExtensionError):
            append_pages(*args)


# ------------------------------------------------------------------------------------------------ planner
def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_plan(tables, ring, counters, lens, new, page, tokens):
    want = R.PlanRef.step(tables.tolist(), ring.tolist(), counters.tolist(), lens.tolist(), new, page, tokens)
    got = plan_pages(tables, ring, counters, lens, ints(new), page, tokens)
    for g, w, name in zip(got, want, ("tables", "ring", "starts", "lens", "counters", "slots")):
        assert g.tolist() == list(w), name
    return got


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("requests", [1, 5, 300, 2500])
def test_plan_pages_steps(page, requests):
    """Twenty steps of growth, single tokens, cuts and ends against the definition: tables, ring, slots, all of them exact."""
    import random

    rng = random.Random(requests)
    width, size = 6, max(8, requests * 3)
    tables, ring, counters, lens = torch.full((requests, width), -1, dtype=torch.int32, device="cuda"), torch.randperm(size).int().cuda(), ints([0, size]), ints([0] * requests)
    for _ in range(20 if requests < 2000 else 4):
        new = [rng.choice((x, x + 1, x + 1, min(x + rng.randint(1, 3 * page), width * page), max(0, x - rng.randint(0, 2 * page)), 0)) for x in lens.tolist()]
        tables, ring, _, lens, counters, _ = check_plan(tables, ring, counters, lens, new, page, requests * 3 * page)


def test_plan_pages_shortage_and_bad_lengths():
    tables, ring = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), ints([3, 1, 0, 2])
    tables, ring, _, lens, counters, _ = check_plan(tables, ring, ints([2, 4]), ints([0, 0, 0]), [20, 30, 0], 16, 64)
    assert counters.tolist()[2] == 0 and lens.tolist() == [20, 30, 0]
    tables, ring, _, lens2, counters2, slots = check_plan(tables, ring, counters, lens, [33, 5, 20], 16, 64)   # three pages wanted, none free
    assert counters2.tolist()[2] == 3 and lens2.tolist() == [20, 5, 0] and (slots == -1).all()
    tables, ring, _, lens3, counters3, _ = check_plan(tables, ring, counters2, lens2, [33, 5, 0], 16, 64)        # the page given back serves now
    assert counters3.tolist()[2] == 0 and lens3.tolist() == [33, 5, 0]
    got = check_plan(tables, ring, counters3, lens3, [33, 10, 0], 16, 4)                                         # slots too short
    assert got[4].tolist()[2] == -1 and got[3].tolist() == [33, 5, 0]
    check_plan(tables, ring, counters3, lens3, [-3, 2 ** 31 - 1, 0], 16, 100)                                   # clamped to the table


def test_plan_pages_again_on_the_same_state_changes_nothing():
    tables, ring, counters, lens = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), ints([5, 4, 3, 2, 1, 0]), ints([4, 6]), ints([0, 0])
    first = [t.clone() for t in plan_pages(tables, ring, counters, lens, ints([40, 17]), 16, 80)]
    again = plan_pages(tables, ring, counters, lens, ints([40, 17]), 16, 80)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_plan_pages_refusals_and_nothing_to_do():
    t, r, c, n = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), ints([0, 1]), ints([0, 2]), ints([0, 0])
    for args in ((t.long(), r, c, n, n, 16, 4), (t, r.long(), c, n, n, 16, 4), (t, r, c[:1], n, n, 16, 4), (t, r, c, n[:1], n, 16, 4), (t, r, c, n, n, 24, 4),
                 (t, r, c, n, n, 16, -1), (t, r.cpu(), c, n, n, 16, 4), (t[:1].expand(2, 4), r, c, n, n, 16, 4), (t.t(), r, c, ints([0] * 4), ints([0] * 4), 16, 4)):
        with pytest.raises(_C.HipExtensionError):
            plan_pages(*args)
    out = plan_pages(t[:0], r, c, n[:0], n[:0], 16, 3)
    assert out[2].tolist() == [0] and out[4].tolist() == [0, 2, 0] and out[5].tolist() == [-1] * 3
    out = plan_pages(t, r[:0], ints([0, 0]), n, n, 16, 0)
    assert out[4].tolist() == [0, 0, 0]


# ------------------------------------------------------------------------------------------------ together
def step(cache, new, x, hq, causal, dims):
    """One step of a scene: plan, write, attend; x: rows of the added tokens [T, (hq + 2 hkv) D]."""
    hkv, dim = dims
    starts, slots = cache.plan(new, x.shape[0])
    q, k, v = (y.unflatten(1, (-1, dim)) for y in x.split([hq * dim, hkv * dim, hkv * dim], 1))
    cache.append(k, v, slots)
    return cache.attend(q, x.shape[0], cache.tables.shape[1] * cache.page, cu_q=starts, causal=causal)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,dim,page", [(4, 4, 64, 64), (8, 2, 128, 16)])
def test_scene_that_grows(dt, hq, hkv, dim, page):
    """Prompts, single tokens, an end and a new request through the cache, every step against attention over what the cache holds; the
    held values against the rows that were written (half an e4m3 step of each, 2^-10 of the scale where it rounds twice)."""
    cache = PagedKVCache(3, 900, 60, hkv, dim, page)
    rows = [torch.zeros(0, 2, hkv, dim, dtype=torch.float64, device="cuda") for _ in range(3)]
    lens = [0, 0, 0]
    for i, new in enumerate([[100, 37, 0], [101, 38, 1], [102, 39, 300], [103, 0, 301], [160, 90, 302], [161, 91, 303]]):
        added = [max(0, b - a) for a, b in zip(lens, new)]
        x = rand((sum(added), (hq + 2 * hkv) * dim), 40 + i, R.H16[dt])
        o = step(cache, ints(new), x, hq, True, (hkv, dim))
        at = 0
        for b in range(3):
            part = x[at:at + added[b], hq * dim:].double().view(added[b], 2, hkv, dim)
            rows[b] = torch.cat([rows[b], part])[:new[b]]
            at += added[b]
        lens = new
        assert cache.lens.tolist() == new and cache.counters.tolist()[2] == 0
        k, v = R.held(cache.pages, cache.tables, lens)
        q = x[:, :hq * dim].unflatten(1, (hq, dim))
        ref = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(ref)
        a, r0 = 0, 0
        for b in range(3):
            if added[b]:
                ref[a:a + added[b]], tol[a:a + added[b]] = R.attention(q[a:a + added[b]], k[r0:r0 + lens[b]], v[r0:r0 + lens[b]], [added[b]], [lens[b]], True)
            a, r0 = a + added[b], r0 + lens[b]
        R.close(o, ref, tol)
        for got, side in ((k, 0), (v, 1)):
            want = torch.cat([r[:, side] for r in rows])
            # the first rounding, and a second one where the scale grew: 2^-4 each; subnormal steps: 2^-10 of a scale <= 2^-5 (|x| < 8)
            assert ((got - want).abs() <= want.abs() * (2 ** -4 + 2 ** -4 * (1 + 2 ** -4)) + 2 * 2.0 ** -15).all()


def test_step_in_a_captured_graph():
    """A decode step captured once and replayed, with eager work between the replays, goes on token by token as eager steps do."""
    hq, hkv, dim = 8, 2, 64
    caches = [PagedKVCache(4, 400, 40, hkv, dim, 16) for _ in range(2)]
    start = rand((75, (hq + 2 * hkv) * dim), 1, torch.float16)
    for c in caches:
        step(c, ints([30, 0, 5, 40]), start, hq, True, (hkv, dim))
    x, new = rand((4, (hq + 2 * hkv) * dim), 2, torch.float16), ints([31, 1, 6, 41])
    keep = [t.clone() for t in (caches[0].lens, caches[0].counters, caches[0].tables, caches[0].ring, *caches[0].pages)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], new, x, hq, True, (hkv, dim))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], new, x, hq, True, (hkv, dim))
    for t, old in zip((caches[0].lens, caches[0].counters, caches[0].tables, caches[0].ring, *caches[0].pages), keep):
        t.copy_(old)
    for i in range(5):
        y = rand(x.shape, 10 + i, torch.float16)
        at = ints([31 + i, 1 + i, 6 + i, 41 + i])
        x.copy_(y), new.copy_(at)
        graph.replay()
        want = step(caches[1], at, y, hq, True, (hkv, dim))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(caches[0].lens, caches[1].lens) and torch.equal(caches[0].pages.k_codes, caches[1].pages.k_codes)


def test_two_captured_graphs_do_not_share_scratch():
    """Two split attentions captured apart and replayed at the same time on two streams give what they give alone."""
    q = [rand((2, 4, 64), 50 + i, torch.float16) for i in range(2)]
    k, v = rand((30000, 1, 64), 60, torch.float16), rand((30000, 1, 64), 61, torch.float16)
    cu_q, cu_k = R.starts([1, 1], "cuda"), R.starts([14000, 16000], "cuda")
    alone = [packed_attention(x, k, v, cu_q, cu_k, 1, 16000) for x in q]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in q]
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(packed_attention(x, k, v, cu_q, cu_k, 1, 16000))
        graphs.append(g)
    for _ in range(3):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, outs))


def test_calls_repeat_bit_for_bit_and_follow_the_current_stream():
    q, k, v = rand((1000, 8, 128), 1, torch.bfloat16), rand((1000, 2, 128), 2, torch.bfloat16), rand((1000, 2, 128), 3, torch.bfloat16)
    cu = R.starts([400, 600], "cuda")
    first = packed_attention(q, k, v, cu, cu, 600, 600)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late = packed_attention(q * 1.0, k, v, cu, cu, 600, 600)
    side.synchronize()
    assert torch.equal(first, late) and torch.equal(first, packed_attention(q, k, v, cu, cu, 600, 600))


# ------------------------------------------------------------------------------------------------ far ends of the ranges
def test_packed_attention_offsets_beyond_32_bits():
    """Keys whose rows lie 32 MB apart: element and byte offsets pass 2^31 and 2^32 (and a stride that a tile could not span is refused)."""
    rows, stride = 200, 2 ** 24 - 8
    buf = torch.zeros(rows * stride + 64, dtype=torch.float16, device="cuda")
    k = buf.as_strided((rows, 1, 64), (stride, 64, 1))
    v = buf.as_strided((rows, 1, 64), (stride, 64, 1), 64)
    k.copy_(rand((rows, 1, 64), 1, torch.float16)), v.copy_(rand((rows, 1, 64), 2, torch.float16))
    q = rand((50, 2, 64), 3, torch.float16)
    o = packed_attention(q, k, v, R.starts([10, 40], "cuda"), R.starts([7, 193], "cuda"), 40, 193)
    R.close(o, *R.attention(q, k, v, [10, 40], [7, 193], True))
    with pytest.raises(_C.HipExtensionError):
        wide = buf.as_strided((100, 1, 64), (2 ** 24, 64, 1))
        packed_attention(q, wide, wide, R.starts([50], "cuda"), R.starts([100], "cuda"), 50, 100)


@pytest.mark.parametrize("rows", [1, 40])
def test_cache_beyond_4_gib(rows):
    """A pool of 4.6 GB of codes: the pages in use are its first and its last ones."""
    total, heads, page, dim = 70000, 16, 64, 64
    pages = Pages.empty(total, heads, dim, page)
    assert pages.k_codes.numel() > 2 ** 32
    ids = [69999, 0, 35001, 69998]
    tables = ints([ids])
    kv = rand((230, 2, heads, dim), 1, torch.float16)
    slots = ints([ids[i // page] * page + i % page for i in range(230)])
    append_pages(pages, kv[:, 0], kv[:, 1], slots)
    q = rand((rows, heads, dim), 2, torch.float16)
    o = paged_attention(q, pages, tables, ints([230]), rows, 230, cu_q=R.starts([rows], "cuda"))
    few = Pages(*(t[ids].contiguous() for t in pages))
    k, v = R.held(few, ints([[0, 1, 2, 3]]), [230])
    R.close(o, *R.attention(q, k, v, [rows], [230], True))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [40, 130])
def test_packed_attention_many_sequences(n, causal):
    """Sequences of 0 to 96 tokens, ranked by length on the GPU (up to 64 of them) or not."""
    lens = [(37 * i) % 97 for i in range(n)]
    run_packed(lens, [max(0, x - 3) if i % 3 else x + 20 for i, x in enumerate(lens)], 3, 3, 64, "bf16", causal, seed=n)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_paged_attention_strided_rows_and_tables(dt):
    """Queries inside a fused matrix, output inside a wider one, tables inside a larger array."""
    lens = [90, 200, 33]
    pages, tables = make_cache(lens, 32, 2, 128, 4)
    wide = torch.full((3, 64), -9, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + tables.shape[1]] = tables
    fused = rand((3, 3, 4, 128), 5, R.H16[dt])
    out = torch.full((3, 4, 256), 7.0, dtype=R.H16[dt], device="cuda")
    o = paged_attention(fused[:, 1], pages, wide[:, 5:5 + tables.shape[1]], ints(lens), 1, 200, out=out[:, :, 128:])
    k, v = R.held(pages, tables, lens)
    R.close(o, *R.attention(fused[:, 1], k, v, [1, 1, 1], lens, True))
    assert (out[:, :, :128] == 7).all()


def test_paged_attention_lengths_beyond_max_len():
    """max_len only chooses the key ranges: a request that holds more is still attended to whole."""
    lens = [9000, 20]
    pages, tables = make_cache(lens, 64, 1, 64, 6)
    q = rand((2, 2, 64), 7, torch.bfloat16)
    k, v = R.held(pages, tables, lens)
    ref, tol = R.attention(q, k, v, [1, 1], lens, True)
    for bound in (9000, 5000, 100, 1):
        R.close(paged_attention(q, pages, tables, ints(lens), 1, bound), ref, tol)


def test_plan_pages_of_8192_requests():
    import random

    rng = random.Random(1)
    n, page, width = 8192, 16, 3
    lens = [rng.randint(0, 48) for _ in range(n)]
    new = [rng.randint(0, 48) for _ in range(n)]
    held = [-(-x // page) for x in lens]
    size = sum(held) + n * 3
    ids = list(range(size))
    rng.shuffle(ids)
    tables, at = [], 0
    for h in held:
        tables.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    ring = [-1] * size
    head = size - 5
    for i, x in enumerate(ids[at:]):
        ring[(head + i) % size] = x
    check_plan(ints(tables), ints(ring), ints([head, size - at]), ints(lens), new, page, n * 48)


def test_cached_values_at_the_edges_of_the_types():
    """fp16: values up to 65 504 (their e4m3 neighbour is 65 536) and down to the subnormals; bf16: 1e30 and 1e-30 in one cache."""
    for dt, sizes in (("f16", (65504.0, 1.0, 3e-5)), ("bf16", (1e30, 1.0, 1e-30))):
        pages = Pages.empty(3, 1, 64, 64)
        k, v = rand((192, 1, 64), 1, R.H16[dt]), rand((192, 1, 64), 2, torch.float32).clamp(-1, 1)
        scale = torch.tensor(sizes, device="cuda").repeat_interleave(64)[:, None, None]
        v = (v * scale).to(R.H16[dt])
        append_pages(pages, k, v, torch.arange(192, dtype=torch.int32, device="cuda"))
        q = rand((20, 1, 64), 3, R.H16[dt])
        for n in (64, 128, 192):     # (the last keys alone decide where large values would hide the small ones)
            tables = ints([[2, 1, 0][:n // 64]])
            kk, vv = R.held(pages, tables, [n])
            for rows in (1, 20):
                o = paged_attention(q[:rows], pages, tables, ints([n]), rows, n, cu_q=R.starts([rows], "cuda"), causal=False)
                R.close(o, *R.attention(q[:rows], kk, vv, [rows], [n], False))


def test_calls_of_more_than_32_bits_are_refused():
    """Expanded operands whose row counts a 32-bit number does not hold."""
    q, cu = rand((8, 2, 64), 1, torch.float16), R.starts([8], "cuda")
    many = q[:1].expand(2 ** 31, 2, 64)
    idx = torch.zeros(4, dtype=torch.int32, device="cuda")
    pages = Pages.empty(2, 2, 64, 16)
    for call in (lambda: packed_attention(q, many, many, cu, cu, 8, 8), lambda: packed_attention(many, q, q, cu, cu, 8, 8),
                 lambda: packed_attention(q, q, q, cu, cu, 8, 8, scale=1e39), lambda: packed_attention(q, q, q, cu, cu, 8, 8, scale=1e-50),
                 lambda: packed_attention(q, q, q, cu, cu, 8, 8, out=torch.zeros_like(q).requires_grad_()),
                 lambda: append_pages(pages, many, many, idx),
                 lambda: plan_pages(idx.view(1, 4), idx, idx, idx[:1], idx[:1], 16, 2 ** 32),
                 lambda: plan_pages(idx.view(1, 4), idx, idx, idx[:1], idx[:1], 16, 2 ** 31 - 1)):
        with pytest.raises(_C.HipExtensionError):
            call()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("dim,lens,keys", [(64, [300, 1, 40], [300, 700, 0]), (128, [300, 1, 40], [300, 700, 0]), (64, [9], [5000]), (64, [2300] * 4, [2300] * 4)])
def test_output_in_the_place_of_the_queries(dt, dim, lens, keys):
    """out = q (a slice of a joint projection too): bit for bit what separate memory gives, packed and from the cache."""
    g = 2
    x = rand((sum(lens), 8 * g, dim), 5, R.H16[dt])
    q = x[:, g:3 * g]
    k, v = rand((sum(keys), g, dim), 6, R.H16[dt]), rand((sum(keys), g, dim), 7, R.H16[dt])
    cu_q, cu_k = R.starts(lens, "cuda"), R.starts(keys, "cuda")
    want = packed_attention(q, k, v, cu_q, cu_k, max(lens), max(keys))
    mine = x.clone()[:, g:3 * g]
    assert packed_attention(mine, k, v, cu_q, cu_k, max(lens), max(keys), out=mine) is mine and torch.equal(mine, want)
    pages, tables = make_cache(keys, 16, g, dim)
    held = torch.tensor(keys, dtype=torch.int32, device="cuda")
    want = paged_attention(q, pages, tables, held, max(lens), max(keys), cu_q=cu_q)
    mine = x.clone()[:, g:3 * g]
    paged_attention(mine, pages, tables, held, max(lens), max(keys), cu_q=cu_q, out=mine)
    assert torch.equal(mine, want)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,lq,page,hq,hkv", [([500, 1, 0, 63, 64, 65, 127, 128, 129, 256] + [200 + i for i in range(30)], [256, 1, 0, 63, 7, 65, 127, 130, 129, 256] + [33] * 30, 16, 16, 16),
                                                 ([1900, 1, 1000, 64, 0, 700], [63, 1, 63, 30, 0, 20], 64, 64, 16), ([2000, 1100, 70], [400, 380, 70], 128, 16, 16)])
def test_paged_attention_of_256_row_tiles_of_64_channels(dt, causal, lens, lq, page, hq, hkv):
    """Two query blocks per wave over 8-bit keys: tiles that end anywhere, empty requests, key ranges, shared heads."""
    run_paged(lens, lq, page, hq, hkv, 64, dt, causal, seed=11)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_attention_of_256_row_tiles_with_bad_pages_and_nan(dt, causal):
    lens, lq, page = [200, 330, 500] + [16] * 37, [256, 256, 256] + [16] * 37, 32
    pages, tables = make_cache(lens, page, 16, 64, 5)
    tables[0, 1], tables[1, 4], tables[1, 0], tables[1, 10] = -1, 10 ** 6, -7, 2 ** 30
    last = int(tables[0, 6])
    pages.v_codes[last, 0, 0, 5, 6] = 0x7f                   # token 198 of request 0
    pages.k_codes[last, 1, 7, 9] = 0xff                      # token 199
    pages.v_codes[int(tables[2, 15]), 3, 0, 7, 1] = 0xff     # token 481 of request 2
    q = rand((sum(lq), 16, 64), 6, R.H16[dt])
    o = paged_attention(q, pages, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), 256, 500, cu_q=R.starts(lq, "cuda"), causal=causal)
    seen = [torch.ones(n, dtype=torch.bool, device="cuda") for n in lens]
    seen[0][32:64] = False
    seen[1][:32] = seen[1][128:160] = seen[1][320:] = False
    k, v = R.held(pages, tables, lens)
    ref, tol = R.attention(q, k, v, lq, lens, causal, seen=seen)
    R.close(o, ref, tol)
