"""64-bit references of the packed-sequence and paged-cache operators, and the error bounds their tests use."""
import math

import torch

H16 = {"bf16": torch.bfloat16, "f16": torch.float16}


def attention(q, k, v, lq, lk, causal, scale=None, seen=None):
    """(o, bound) of packed sequences of lq rows and lk keys in float64; q [Tq, Hq, D], k and v [Tk, Hkv, D].  seen[b] [lk]: keys that
    exist (default all).  `bound` is how far a kernel with 16-bit operands may be off, entry by entry, for h = half a step of the
    operand type (relative), A = sum_j p_j |v_j|:
        h |o|                     the output's rounding,
        h A                       the numerators' rounding before the second product,
        2 (D + 8) u S A           fp32 accumulation of a score (u = 2^-24, S = scale sum_d |q_d k_d|, the largest of the row) and the
                                  exponential, as a relative error of p and of the row sum,
        (2 N + 64) u A            fp32 accumulation of O and l over N keys,
        2^-24 + N 2^-32 max |v|   fp16's subnormal steps: of the output and the halved 8-bit values, of the numerators (8 bits above
                                  the largest one, less 4 that the maximum may lag)"""
    hq, hkv, dim = q.shape[1], k.shape[1], q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    h, u = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    qd, kd, vd = q.double(), k.double(), v.double()
    r0 = k0 = 0
    for b, (n, m) in enumerate(zip(lq, lk)):
        for head in range(hq):
            if n == 0 or m == 0:
                continue
            qq, kk, vv = qd[r0:r0 + n, head], kd[k0:k0 + m, head * hkv // hq], vd[k0:k0 + m, head * hkv // hq]
            mask = torch.ones(n, m, dtype=torch.bool, device=q.device)
            if causal:
                mask = torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + (m - n)
            if seen is not None:
                mask = mask & seen[b][None]
            s = torch.where(mask, scale * (qq @ kk.t()), -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(mask, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            o = torch.where(mask[..., None], p[..., None] * vv[None], 0.0).sum(1) if not vv.isfinite().all() else p @ vv
            out[r0:r0 + n, head] = o
            a = p @ vv.abs().nan_to_num(0.0, 0.0, 0.0)
            big = torch.where(mask, scale * (qq.abs() @ kk.abs().t()), 0.0).nan_to_num(0.0, 0.0, 0.0).amax(-1, keepdim=True)
            tol[r0:r0 + n, head] = (h * o.abs() + (h + 2 * (dim + 8) * u * big + (2 * m + 64) * u) * a + 2.0 ** -24
                                    + m * 2.0 ** -32 * vv.abs().nan_to_num(0.0, 0.0, 0.0).amax())
        r0, k0 = r0 + n, k0 + m
    return out, tol


def close(got, ref, tol):
    """Asserts |got - ref| <= tol where ref is finite, and the same infinities and NaN elsewhere."""
    got = got.double()
    fine = ref.isfinite()
    assert torch.equal(fine, got.isfinite()), "finite entries differ"
    assert torch.equal(ref.isnan(), got.isnan()), "NaN entries differ"
    inf = ref.isinf()
    assert torch.equal(ref[inf], got[inf]), "infinities differ"
    over = (got - ref)[fine].abs() - tol[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"off by {float((got - ref)[fine].abs().max()):.3e}, {float(over.max()):.3e} over the bound"


def starts(lengths, device="cpu"):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=device)


def e4m3(x):
    """Nearest e4m3 value of float64 x (ties to even, +-448 at most, NaN stays)."""
    y = x.clamp(-448.0, 448.0)
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))).clamp(-6, 8)
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


class CacheRef:
    """The cache as float64 values of codes and integer exponents, by the definition (one page and head at a time)."""

    def __init__(self, pages, heads, page, dim):
        self.page = page
        self.code = [torch.zeros(pages, heads, page, dim, dtype=torch.float64) for _ in range(2)]
        self.byte = [torch.zeros(pages, heads, dtype=torch.int64) for _ in range(2)]

    def append(self, k, v, slots):
        t = 0
        total = self.code[0].shape[0] * self.page
        while t < len(slots):
            s = slots[t]
            if not 0 <= s < total:
                t += 1
                continue
            n = 1
            while t + n < len(slots) and slots[t + n] == s + n and (s + n) % self.page:
                n += 1
            for side, x in enumerate((k, v)):
                self._run(side, s // self.page, s % self.page, x[t:t + n].double().cpu())
            t += n

    def _run(self, side, page, at, x):
        for head in range(x.shape[1]):
            y = x[:, head]
            amax = float(torch.where(y.isfinite(), y.abs(), 0.0).max())
            need = 1
            if amax > 0:
                m, e = math.frexp(amax)                       # 448 = 0.875 * 2^9
                need = min(max(e - 9 + (m > 0.875) + 127, 1), 254)
            old = int(self.byte[side][page, head])
            now = max(old, need) if at else need
            if at and now > old:
                self.code[side][page, head, :at] = e4m3(self.code[side][page, head, :at] * 2.0 ** (old - now))
            self.code[side][page, head, at:at + x.shape[0]] = e4m3(y * 2.0 ** (127 - now))
            self.byte[side][page, head] = now


def code_values(pages):
    """(K, V) codes of a Pages tuple as float64 [pages, heads, page, dim] on the CPU."""
    n, h, page, dim = pages.k_codes.shape
    k = pages.k_codes.cpu().view(torch.float8_e4m3fn).double()
    v = pages.v_codes.cpu().view(torch.float8_e4m3fn).double().permute(0, 1, 2, 4, 3).reshape(n, h, page, dim)
    return k, v


def held(pages, tables, lens):
    """K and V rows [sum lens, heads, dim] (float64, on the device) that the cache stands for."""
    n, h, page, dim = pages.k_codes.shape
    dev = pages.k_codes.device
    ks, vs = [], []
    k, v = (x.to(dev) for x in code_values(pages))
    k = k * torch.exp2(pages.k_scale.double() - 127)[:, :, None, None]
    v = v * torch.exp2(pages.v_scale.double() - 127)[:, :, None, None]
    for b, m in enumerate(lens):
        t = torch.arange(m, device=dev)
        ids = tables[b].long()[t // page].clamp(0, n - 1)
        ks.append(k[ids, :, t % page]), vs.append(v[ids, :, t % page])
    return torch.cat(ks), torch.cat(vs)


class PlanRef:
    """The planner by its definition, with a Python list of free pages."""

    @staticmethod
    def step(tables, ring, counters, lens, new_lens, page, tokens):
        tables, ring = [list(r) for r in tables], list(ring)
        size, width = len(ring), len(tables[0]) if tables else 0
        head, count = counters[0], counters[1]
        cap = width * page
        have, want = [min(max(x, 0), cap) for x in lens], [min(max(x, 0), cap) for x in new_lens]
        pages = lambda n: -(-n // page)  # noqa: E731
        grow = sum(max(0, pages(w) - pages(h)) for h, w in zip(have, want))
        added = sum(max(0, w - h) for h, w in zip(have, want))
        missing = -1 if added > tokens else max(0, grow - count)
        tail, freed = head + count, 0
        slots, starts_, out = [], [0], []
        before = [list(r) for r in tables]
        for b, (h, w) in enumerate(zip(have, want)):
            if w < h:
                for j in range(pages(w), pages(h)):
                    ring[(tail + freed) % size] = before[b][j]
                    freed += 1
            elif missing == 0:
                for j in range(pages(h), pages(w)):
                    tables[b][j] = ring[head % size]
                    head, count = head + 1, count - 1
                slots += [tables[b][t // page] * page + t % page for t in range(h, w)]
            out.append(w if w < h or missing == 0 else h)
            starts_.append(len(slots))
        slots += [-1] * (tokens - len(slots))
        return tables, ring, starts_, out, [head % size, count + freed, missing], slots
