"""CPU checks of the packed-sequence and paged-cache operators: refusals before any launch, and the references against plain
formulas (the kernels themselves: test_packed_gpu.py)."""
import ctypes
import struct

import pytest
import torch

import packed_ref as R
from iggt_official_amd import _C
from iggt_official_amd.layers import packed as P


@pytest.fixture(scope="module")
def lib():
    from iggt_official_amd import build_ext

    build_ext.build(verbose=False)
    return _C.load()


def _packed(lib, **kw):
    a = dict(q=16, q_rs=64, q_hs=64, k=16, k_rs=64, k_hs=64, v=16, v_rs=64, v_hs=64, o=16, o_rs=64, o_hs=64, cu_q=16, cu_k=16, B=0, Tq=4, Tk=4,
             max_q=4, max_k=4, Hq=1, Hkv=1, D=64, scale=1.0, causal=1, ws=0, ws_len=0, stream=0)
    a.update(kw)
    return lib.iggt_packed_attn_bf16(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(D=96), -1), (dict(Hq=3, Hkv=2), -1), (dict(B=-1), -1), (dict(q_rs=60), -2), (dict(k_hs=4), -2), (dict(q=8), -2),
                                   (dict(o=4), -2), (dict(scale=0.0), -3), (dict(scale=float("nan")), -3),
                                   (dict(B=1, Tq=1, Tk=100000, max_q=1, max_k=100000), -5), (dict(), 0)])
def test_packed_entry_refuses_on_the_host(lib, kw, rc):
    """Negative codes come before any launch (B = 0: nothing to do)."""
    assert _packed(lib, **kw) == rc


def _paged(lib, **kw):
    a = dict(q=16, q_rs=64, q_hs=64, o=16, o_rs=64, o_hs=64, kc=16, ks=16, vc=16, vs=16, pages=4, page=64, tables=16, stride=4, width=4, lens=16,
             cu_q=16, B=0, Tq=4, max_q=4, max_len=4, Hq=1, Hkv=1, D=64, scale=1.0, causal=1, ws=0, ws_len=0, stream=0)
    a.update(kw)
    return lib.iggt_paged_attn_f16(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(page=48), -1), (dict(D=32), -1), (dict(cu_q=0), -1), (dict(width=1 << 26), -1), (dict(Hq=5, Hkv=2), -1),
                                   (dict(kc=8), -2), (dict(q_hs=9), -2), (dict(scale=-1.0), -3),
                                   (dict(B=1, max_q=1, max_len=100000), -5), (dict(), 0)])
def test_paged_entry_refuses_on_the_host(lib, kw, rc):
    assert _paged(lib, **kw) == rc


def test_writer_and_planner_entries_refuse_on_the_host(lib):
    ap = lambda **kw: lib.iggt_append_pages_bf16(*{**dict(k=16, k_rs=64, k_hs=64, v=16, v_rs=64, v_hs=64, slots=16, T=0, kc=16, ks=16, vc=16, vs=16,  # noqa: E731
                                                         pages=4, page=64, H=1, D=64, stream=0), **kw}.values())
    assert ap() == 0 and ap(page=63) == -1 and ap(D=72) == -1 and ap(k_rs=12) == -2 and ap(v=8) == -2 and ap(pages=1 << 26) == -1
    pl = lambda **kw: lib.iggt_plan_pages(*{**dict(tables=16, stride=4, R=1, M=4, ring=16, N=4, counters=16, lens=16, new=16, page=64, starts=16,  # noqa: E731
                                                   nl=16, nc=16, slots=16, T=4, stream=0), **kw}.values())
    assert pl(R=8193) == -1 and pl(page=20) == -1 and pl(T=-1) == -1 and pl(M=1 << 25) == -1 and pl(N=1 << 26) == -1


def test_workspace_sizes_follow_the_key_ranges(lib):
    """No scratch where the grid fills the chip, (D + 2) floats per row and range where it does not."""
    assert lib.iggt_packed_attn_ws_bytes(32, 2000, 2000, 16, 16, 64) == 0
    n = lib.iggt_packed_attn_ws_bytes(1, 1, 100000, 16, 16, 64)
    assert n > 0 and n % (16 * 66 * 4) == 0
    assert lib.iggt_paged_attn_ws_bytes(1, 1, 256, 16, 16, 64) == 0
    assert lib.iggt_paged_attn_ws_bytes(1, 1, 100000, 16, 16, 128) % (16 * 130 * 4) == 0
    assert lib.iggt_packed_attn_ws_bytes(1, 1, 100000, 3, 2, 64) == 0


def test_cpu_tensors_are_refused():
    z = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    pages = P.Pages.empty(2, 2, 64, 16, "cpu")
    with pytest.raises(_C.HipExtensionError):
        P.packed_attention(z, z, z, i, i, 4, 4)
    with pytest.raises(_C.HipExtensionError):
        P.paged_attention(z, pages, i.view(1, 2), i[:1], 4, 4, cu_q=i)
    with pytest.raises(_C.HipExtensionError):
        P.append_pages(pages, z, z, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(_C.HipExtensionError):
        P.plan_pages(i.view(1, 2), i, i, i[:1], i[:1], 16, 4)
    for bad in (dict(page=24), dict(head_dim=80), dict(requests=0), dict(longest=0)):
        with pytest.raises(_C.HipExtensionError):
            P.PagedKVCache(**{**dict(requests=1, longest=64, pages=2, kv_heads=1, head_dim=64, page=16, device="cpu"), **bad})


def test_reference_attention_is_softmax_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(9, 4, 64, generator=g).bfloat16(), torch.randn(13, 2, 64, generator=g).bfloat16(), torch.randn(13, 2, 64, generator=g).bfloat16())
    o, _ = R.attention(q, k, v, [4, 0, 5], [6, 4, 3], True)
    kk, vv = k.double().repeat_interleave(2, 1), v.double().repeat_interleave(2, 1)
    for r0, n, k0, m in ((0, 4, 0, 6), (4, 5, 10, 3)):
        s = torch.einsum("qhd,khd->hqk", q[r0:r0 + n].double(), kk[k0:k0 + m]) / 8
        s = s.masked_fill(torch.ones(n, m).tril(m - n) == 0, float("-inf"))
        ref = torch.einsum("hqk,khd->qhd", s.softmax(-1).nan_to_num(0.0), vv[k0:k0 + m])
        assert torch.allclose(o[r0:r0 + n], ref, atol=1e-12)
    assert (o[4:6] == 0).all()      # 5 rows, 3 keys: the first two see none


def test_reference_codes_are_torchs_e4m3():
    x = torch.cat([torch.linspace(-460, 460, 4001), torch.linspace(-0.05, 0.05, 4001)]).double()
    assert torch.equal(R.e4m3(x).float(), x.clamp(-448, 448).float().to(torch.float8_e4m3fn).float())


def test_reference_planner_keeps_every_page_once():
    import random

    rng = random.Random(3)
    page, width, n, size = 16, 8, 5, 24
    tables, ring, counters, lens = [[-1] * width for _ in range(n)], list(range(size)), [0, size, 0], [0] * n
    for _ in range(60):
        new = [rng.choice((0, x, min(x + rng.randint(0, 40), width * page), max(0, x - 20))) for x in lens]
        tables, ring, _, lens, counters, _ = R.PlanRef.step(tables, ring, counters, lens, new, page, 200)
        out = [tables[b][j] for b in range(n) for j in range(-(-lens[b] // page))]
        free = [ring[(counters[0] + i) % size] for i in range(counters[1])]
        assert sorted(out + free) == list(range(size))


def test_sizes_beyond_32_bits_are_refused_on_the_host(lib):
    """Counts whose products or whose next step would pass 2^31: before any launch."""
    assert _packed(lib, B=1, Tq=1 << 21, Hq=1 << 10, Hkv=1) == -1 and _paged(lib, B=1, Tq=1 << 21, Hq=1 << 10, Hkv=1) == -1
    assert _packed(lib, scale=3e38) == -3 and _paged(lib, scale=float("inf")) == -3
    plan = lambda R, M, T: lib.iggt_plan_pages(16, M, R, M, 16, 4, 16, 16, 16, 16, 16, 16, 16, 16, T, 0)  # noqa: E731
    assert plan(8192, 1 << 18, 4) == -1 and plan(1, 4, 0x7fffffff) == -1
    assert lib.iggt_append_pages_f16(16, 64, 64, 16, 64, 64, 16, 0x7fffffff, 16, 16, 16, 16, 4, 64, 1, 64, 0) == -1


def test_calls_with_arguments_in_memory(lib):
    """iggt_seq_call hands every argument to the call that the first word names: the same refusals, one wrong argument at a time."""
    good = dict(packed=(16, 64, 64, 16, 64, 64, 16, 64, 64, 16, 64, 64, 16, 16, 0, 4, 4, 4, 4, 1, 1, 64, 1.0, 1, 0, 0, 0),
                paged=(16, 64, 64, 16, 64, 64, 16, 16, 16, 16, 4, 64, 16, 4, 4, 16, 16, 0, 4, 4, 4, 1, 1, 64, 1.0, 1, 0, 0, 0),
                append=(16, 64, 64, 16, 64, 64, 16, 0, 16, 16, 16, 16, 4, 64, 1, 64, 0), plan=(16, 4, 8193, 4, 16, 4, 16, 16, 16, 64, 16, 16, 16, 16, 4, 0))
    for layout, op, name, key in ((P._PACKED, 0, "iggt_packed_attn_bf16", "packed"), (P._PACKED, 1, "iggt_packed_attn_f16", "packed"),
                                  (P._PAGED, 2, "iggt_paged_attn_bf16", "paged"), (P._PAGED, 3, "iggt_paged_attn_f16", "paged"),
                                  (P._APPEND, 4, "iggt_append_pages_bf16", "append"), (P._APPEND, 5, "iggt_append_pages_f16", "append"),
                                  (P._PLAN, 6, "iggt_plan_pages", "plan")):
        args, codes = good[key], set()
        assert struct.calcsize(layout.format) == 8 * (len(args) + 1)
        for i in range(len(args)):
            for wrong in (-1, 3):
                if key == "plan" and i == 2 or key != "plan" and args[i] == 0 and i in (7, 14, 17):
                    continue                            # these keep the call from a launch
                a = args[:i] + (type(args[i])(wrong),) + args[i + 1:]
                codes.add(lib.iggt_seq_call(layout.pack(op, *a)))
                assert lib.iggt_seq_call(layout.pack(op, *a)) == getattr(lib, name)(*a), (name, i, wrong)
        assert -1 in codes
    assert lib.iggt_seq_call(P._PLAN.pack(7, *good["plan"])) == -1
