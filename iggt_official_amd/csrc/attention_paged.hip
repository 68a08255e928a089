// Attention over a paged K/V cache held in 8 bits (e4m3 codes, one power-of-two scale per page and key head): few query rows per
// request (single tokens, drafts), split over the keys; the fold of key ranges; and the dispatcher, which sends many rows per
// request to the tile kernel of attention_packed.hip.
//
// Few rows: the bound is the read of the codes, 2 D bytes per key and key head.  A wave takes 64 keys at a time straight from
// memory into registers -- no LDS, no barrier in the loop -- and the layouts are chosen so that every load is 16 bytes a lane and
// nothing crosses lanes between load and matrix instruction (16 x 16 x 32, A = keys / channels, B = the up to 16 query rows):
//   S^T:  row a of score tile t (t = 0 .. 3) is key 16 (a >> 2) + 4 t + (a & 3): lane group g = lane >> 4 then holds the scores of keys
//         16 g .. 16 g + 15 of its query row, in order 4 t + r.  A lane's 16 bytes of K are channels 16 g .. 16 g + 15 of one key (two
//         contraction steps); the query fragments use the same channel order.
//   O^T:  the B operand of step u is the lane's own numerators 8 u .. 8 u + 7, so V^T must give lane (d, g) keys 16 g + 8 u ..: the cache
//         keeps 16 keys of a channel side by side, one 16-byte load for both steps.
// Scores are scaled by the page's 2^e in fp32; V is converted with its scale.  The next keys' K codes are loaded while this block's
// softmax runs.  The four waves of a workgroup take every fourth block of its key range and are joined in LDS.
// Measured (MI355X, a large copy moves 5.2 TB/s): one row, 350 784 tokens, 16 heads of 64: 123 us, 5.8 TB/s, + 5 us fold; 64 requests of
// up to 8 192 tokens, 16 query and 4 key heads of 128: 60 us, 4.8 TB/s, + 5 us; one request of 1 374 tokens, 16 heads of 64, not split:
// 7.5 - 8.5 us, the latency of five dependent loads and six blocks per wave.
#include "seq_attention.h"
#include "../../include/iggt_hip.h"

using namespace iggt_seq;

namespace {

template <int FMT>
IGGT_DEVINL f32x4 mfma16h(bf16x8 a, bf16x8 b, f32x4 c) {
    if (FMT == FMT_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// DRAFT: several tokens per request, so that near the end a key may be seen by some rows only.
template <int D, int FMT, bool DRAFT>
__global__ __launch_bounds__(256, DRAFT ? 2 : 3) void seq_attn_rows_kernel(const SeqAttnParams p) {
    constexpr int NC = D / 64, NDT = D / 16;
    constexpr float HALF = FMT == FMT_F16 ? 0.5f : 1.0f;   // fp16 holds half of V's values (a code at the top of its range is 2^16)
    __shared__ float s_o[4][16][D + 4];
    __shared__ float s_ml[4][16][2];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int npairs = p.B * p.Hkv;
    // (the 16-row tiles of one pair and key range lie npairs work items apart: with a multiple of 8 pairs on one XCD, and in any case
    // together in time, so that the codes come from memory once)
    const unsigned item = seq_item();
    const int pair = item % npairs, rest = item / npairs;
    const int row0 = rest % p.qtiles * 16, split = rest / p.qtiles;
    const int b = pair / p.Hkv, h = pair - b * p.Hkv;
    const SeqSpan sp = seq_span<true>(p, b);
    const int rows = min(sp.lq * p.G - row0, 16);
    if (item >= p.items || rows <= 0) return;   // (asked late: the arguments come in one go)
    const int first = p.causal ? max(min(sp.lk, sp.off + row0 / p.G + 1), 0) : sp.lk;    // keys that every row sees
    // keys that some row sees (one token: the same)
    const int kend = !DRAFT ? first : (p.causal ? max(min(sp.lk, sp.off + (row0 + rows - 1) / p.G + 1), 0) : sp.lk);
    // key range of the work item: whole rounds of the four waves (256 keys), of the same length for every request
    const int b0 = split * p.range_blocks;
    const int b1 = split == p.splits - 1 ? (kend + 63) >> 6 : min(b0 + p.range_blocks, (kend + 63) >> 6);   // (max_len may be too small)

    const int rn = row0 + min(n, rows - 1), qi = rn / p.G, hq = h * p.G + rn - qi * p.G;
    const int lim = p.causal ? max(min(sp.lk, sp.off + qi + 1), 0) : sp.lk;
    bf16x8 qf[NC][2];
    {
        const bf16_t* src = p.q + (long)(sp.q0 + qi) * p.q_rs + (long)hq * p.q_hs + 16 * g;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) qf[c][u] = *reinterpret_cast<const bf16x8*>(src + 64 * c + 8 * u);
    }
    f32x4 o[NDT];
#pragma unroll
    for (int i = 0; i < NDT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = M_INIT, l = 0.f;

    const int pmask = (1 << p.page_shift) - 1;
    const int a_sub = n >> 2, a_key = n & 3;
    u32x4 kc[4][NC], vc[NDT];
    // Loads complete in the order they are issued, so nothing may wait for one that is younger than what is meant to stay in flight:
    // page ids are loaded two blocks ahead, the scales in front of the K codes of their block.
    int kp = 0, vp = 0, kp1 = 0, vp1 = 0;          // table entries of the lane's K rows / of its V keys: this block, the next one
    uint32_t kb = 127, vb = 127;                   // their scale bytes, of the group g whose scores the lane holds
    auto pages = [&](int blk, int& k_page, int& v_page) {
        k_page = page_entry(p, b, blk * 64 + a_sub * 16);
        v_page = page_entry(p, b, blk * 64 + g * 16);
    };
    auto load_k = [&](int blk, int k_page, int v_page) {
        const long sidx = (long)(page_ok(p, v_page) ? v_page : 0) * p.Hkv + h;
        kb = p.k_scale[sidx];
        vb = p.v_scale[sidx];
        const uint8_t* src = p.k8 + (((((long)(page_ok(p, k_page) ? k_page : 0) * p.Hkv + h) << p.page_shift) + ((blk * 64 + a_sub * 16) & pmask) + a_key) * D) + 16 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) kc[t][c] = *reinterpret_cast<const u32x4*>(src + (4 * t) * D + 64 * c);
    };
    auto load_v = [&](int blk, int page) {
        const uint8_t* src = p.v8 + (((((long)(page_ok(p, page) ? page : 0) * p.Hkv + h) << p.page_shift) + ((blk * 64 + g * 16) & pmask)) * D) + n * 16;
#pragma unroll
        for (int i = 0; i < NDT; ++i) vc[i] = *reinterpret_cast<const u32x4*>(src + 256 * i);
    };

    int blk = b0 + wave;
    if (blk < b1) {
        pages(blk, kp, vp);
        pages(blk + 4, kp1, vp1);
        load_k(blk, kp, vp);
    }
    for (; blk < b1; blk += 4) {
        load_v(blk, vp);
        const float ks = scale_of(kb) * p.scale_log2, vs = scale_of(vb) * HALF;
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                bf16x8 lo, hi;
                cvt16<FMT>(kc[t][c], 1.0f, lo, hi);
                s[t] = mfma16h<FMT>(lo, qf[c][0], s[t]);
                s[t] = mfma16h<FMT>(hi, qf[c][1], s[t]);
            }
        }
        const int here = vp, kp0 = kp;
        kp = kp1;
        vp = vp1;
        // (the last block loads itself again: with a branch here every later wait would be one for all loads)
        const int next = blk + 4 < b1 ? blk + 4 : blk;
        if (blk + 4 >= b1) {
            kp = kp0;
            vp = here;
        }
        pages(blk + 8, kp1, vp1);
        load_k(next, kp, vp);

        float e[16];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) e[4 * t + r] = s[t][r] * ks;
        const int key0 = blk * 64 + g * 16;
        const bool edge = blk * 64 + 64 > first || __any(!page_ok(p, here));
        const int seen = !page_ok(p, here) ? 0 : lim - key0;       // of the lane's 16 keys, the first `seen` count for its row
        if (edge) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j >= seen) e[j] = -INFINITY;
        }
        float mx = e[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mx = fmaxf(mx, e[j]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NDT; ++i) o[i] *= alpha;
        }
        const float ms = m - (FMT == FMT_F16 ? P_SHIFT_F16 : 0.f);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            e[j] = __builtin_amdgcn_exp2f(e[j] - ms);
            l += e[j];
        }
        const bf16x8 p0 = pack8f<FMT>(e), p1 = pack8f<FMT>(e + 8);
        // 0 * NaN and 0 * inf are NaN: what lies behind the last key that a row sees (whatever the page holds there) is zeroed, and what only
        // some rows see is looked for here -- codes 0x7f / 0xff (NaN; e4m3 has no infinity), and scales at which fp16 does not hold 448
        bool bad = false;
        if (edge) {
            const int held = !page_ok(p, here) ? 0 : kend - key0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int keep = min(max(held - 4 * w, 0), 4);
                const uint32_t bytes = keep == 4 ? ~0u : (1u << (8 * keep)) - 1u;
                uint32_t nan = 0;
#pragma unroll
                for (int i = 0; i < NDT; ++i) {
                    vc[i][w] &= bytes;
                    if (DRAFT) nan |= ((vc[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                }
                if (DRAFT) bad = bad || nan != 0;
            }
            if (DRAFT && FMT == FMT_F16) bad = bad || (vs > 128.f && held > 0);
            if (DRAFT) bad = __any(bad);
        }
        if (!DRAFT || !bad) {
#pragma unroll
            for (int i = 0; i < NDT; ++i) {
                bf16x8 lo, hi;
                cvt16<FMT>(vc[i], vs, lo, hi);
                o[i] = mfma16h<FMT>(lo, p0, o[i]);
                o[i] = mfma16h<FMT>(hi, p1, o[i]);
            }
        } else {
            // the product runs on zeros in the place of values that are not finite; further ones, of 1 where such a value is not negative
            // and of 1 where it is (a NaN: both) with the mask, find the rows that see one
            float one[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) one[j] = j < seen ? 1.f : 0.f;
            const bf16x8 i0 = pack8f<FMT>(one), i1 = pack8f<FMT>(one + 8);
#pragma unroll
            for (int i = 0; i < NDT; ++i) {
                bf16x8 v[2];
                cvt16<FMT>(vc[i], vs, v[0], v[1]);
                f32x4 plus = {0.f, 0.f, 0.f, 0.f}, minus = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    constexpr uint32_t M = FMT == FMT_F16 ? 0x03ff03ffu : 0x007f007fu, ONE = FMT == FMT_F16 ? 0x3c003c00u : 0x3f803f80u;
                    u32x4 w = __builtin_bit_cast(u32x4, v[u]), up, down;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t odd = nonfinite2<FMT>(w[j]);                                  // bits 15 and 31
                        const uint32_t nan = odd & (((w[j] & M) + M) << (FMT == FMT_F16 ? 5 : 8));   // mantissa not 0
                        up[j] = (((odd & ~w[j]) | nan) >> 15) * 0xffffu & ONE;
                        down[j] = (((odd & w[j]) | nan) >> 15) * 0xffffu & ONE;
                        w[j] &= ~((odd >> 15) * 0xffffu);
                    }
                    plus = mfma16h<FMT>(__builtin_bit_cast(bf16x8, up), u ? i1 : i0, plus);
                    minus = mfma16h<FMT>(__builtin_bit_cast(bf16x8, down), u ? i1 : i0, minus);
                    o[i] = mfma16h<FMT>(__builtin_bit_cast(bf16x8, w), u ? p1 : p0, o[i]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (plus[r] > 0.f) o[i][r] += INFINITY;
                    if (minus[r] > 0.f) o[i][r] -= INFINITY;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // ---- join the four waves
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
        s_ml[wave][n][0] = m;
        s_ml[wave][n][1] = l;
    }
#pragma unroll
    for (int i = 0; i < NDT; ++i) *reinterpret_cast<f32x4*>(&s_o[wave][n][16 * i + 4 * g]) = o[i];
    __syncthreads();
    constexpr int LPR = D / 4;   // lanes of a row, four channels each
    for (int r = tid / LPR; r < rows; r += 256 / LPR) {
        const int d = (tid % LPR) * 4;
        float mm = s_ml[0][r][0];
#pragma unroll
        for (int w = 1; w < 4; ++w) mm = fmaxf(mm, s_ml[w][r][0]);
        float ll = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (s_ml[w][r][1] == 0.f) continue;
            const float f = __builtin_amdgcn_exp2f(s_ml[w][r][0] - mm);
            ll += s_ml[w][r][1] * f;
            acc += *reinterpret_cast<const f32x4*>(&s_o[w][r][d]) * f;
        }
        const int i = (row0 + r) / p.G, hr = h * p.G + row0 + r - i * p.G;
        if (p.splits > 1) {
            const long at = (((long)split * p.B + b) * p.max_q + i) * p.Hq + hr;
            if (d == 0) {
                p.part_ml[2 * at] = mm;
                p.part_ml[2 * at + 1] = ll;
            }
            if (ll != 0.f) *reinterpret_cast<f32x4*>(p.part_o + at * D + d) = acc;
        } else {
            const float inv = ll == 0.f ? 0.f : (1.0f / HALF) / ll;
            u32x2 w;
            w[0] = pack_h2<FMT, false>(acc[0] * inv, acc[1] * inv);
            w[1] = pack_h2<FMT, false>(acc[2] * inv, acc[3] * inv);
            *reinterpret_cast<u32x2*>(p.o + (long)(sp.q0 + i) * p.o_rs + (long)hr * p.o_hs + d) = w;
        }
    }
}

// o = sum_s w_s O_s / sum_s w_s l_s, w_s = 2^(m_s - M), over up to FOLD_MAX key ranges.  W waves share a row (four where there are few
// rows: the loads of a row are then a chain of a few); a wave's lanes hold the weights of all ranges, D / 4 lanes take four channels
// of one range each.
template <int D, int FMT, bool PAGED, int W>
__global__ __launch_bounds__(256) void seq_attn_fold_kernel(const SeqAttnParams p) {
    constexpr int LPR = D / 4, NG = 64 / LPR;
    constexpr float HALF = (PAGED && FMT == FMT_F16) ? 0.5f : 1.0f;
    __shared__ f32x4 s_acc[4][LPR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, gr = lane / LPR, d = (lane % LPR) * 4;
    const long row = (long)blockIdx.x * (4 / W) + wave / W;    // ((b, token), head)
    const long per = (long)p.max_q * p.Hq;
    const int b = (int)(row / per);
    SeqSpan sp = {0, 0, 0, 0, 0};
    if (b < p.B) sp = seq_span<PAGED>(p, b);
    const int i = (int)((row - b * per) / p.Hq), hq = (int)(row % p.Hq);
    const bool live = b < p.B && i < sp.lq;
    const long step = (long)p.B * per;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    if (live) {
        static_assert(FOLD_MAX == 64, "a lane for every range");
        float m = M_INIT, l = 0.f;
        if (lane < p.splits) {
            m = p.part_ml[2 * (lane * step + row)];
            l = p.part_ml[2 * (lane * step + row) + 1];
        }
        float top = m;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        const float weight = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - top);
        total = wave_sum(l * weight);
        // (a range without a key has left no sum; one whose weight vanishes counts with 0, so that its infinities and NaN do not get lost)
        const unsigned long long some = __ballot(l != 0.f);
        for (int s = (wave % W) * NG; s < p.splits; s += NG * W) {
            const float f = __shfl(weight, s + gr, 64);
            if ((some >> (s + gr)) & 1) acc += *reinterpret_cast<const f32x4*>(p.part_o + ((s + gr) * step + row) * D + d) * f;
        }
#pragma unroll
        for (int x = LPR; x < 64; x *= 2)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor(acc[j], x, 64);
    }
    if constexpr (W == 4) {
        if (gr == 0) s_acc[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && gr == 0) acc = (s_acc[0][lane] + s_acc[1][lane]) + (s_acc[2][lane] + s_acc[3][lane]);
    }
    if (live && gr == 0 && wave % W == 0) {
        const float inv = total == 0.f ? 0.f : (1.0f / HALF) / total;
        u32x2 w;
        w[0] = pack_h2<FMT, false>(acc[0] * inv, acc[1] * inv);
        w[1] = pack_h2<FMT, false>(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<u32x2*>(p.o + (long)(sp.q0 + i) * p.o_rs + (long)hq * p.o_hs + d) = w;
    }
}

// The same for up to 8 ranges: a thread folds four channels of a row by itself, all its loads independent.
template <int D, int FMT, bool PAGED>
__global__ __launch_bounds__(256) void seq_attn_fold_few_kernel(const SeqAttnParams p) {
    constexpr int LPR = D / 4;
    constexpr float HALF = (PAGED && FMT == FMT_F16) ? 0.5f : 1.0f;
    const int d = (int)(threadIdx.x % LPR) * 4;
    const long row = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;    // ((b, token), head)
    const long per = (long)p.max_q * p.Hq;
    const int b = (int)(row / per);
    if (b >= p.B) return;
    const SeqSpan sp = seq_span<PAGED>(p, b);
    const int i = (int)((row - b * per) / p.Hq), hq = (int)(row % p.Hq);
    if (i >= sp.lq) return;
    const long step = (long)p.B * per;
    float m[8], l[8], top = M_INIT;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        m[s] = M_INIT;
        l[s] = 0.f;
        if (s < p.splits) {
            m[s] = p.part_ml[2 * (s * step + row)];
            l[s] = p.part_ml[2 * (s * step + row) + 1];
        }
        top = fmaxf(top, m[s]);
    }
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        if (s < p.splits && l[s] != 0.f) {
            const float f = __builtin_amdgcn_exp2f(m[s] - top);
            total += l[s] * f;
            acc += *reinterpret_cast<const f32x4*>(p.part_o + (s * step + row) * D + d) * f;
        }
    }
    const float inv = total == 0.f ? 0.f : (1.0f / HALF) / total;
    u32x2 w;
    w[0] = pack_h2<FMT, false>(acc[0] * inv, acc[1] * inv);
    w[1] = pack_h2<FMT, false>(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<u32x2*>(p.o + (long)(sp.q0 + i) * p.o_rs + (long)hq * p.o_hs + d) = w;
}

template <int D, int FMT, bool PAGED>
int launch_fold(const SeqAttnParams& p, hipStream_t stream) {
    const long rows = (long)p.B * p.max_q * p.Hq;
    if (rows >= (1L << 31)) return -4;
    if (p.splits <= 8) hipLaunchKernelGGL((seq_attn_fold_few_kernel<D, FMT, PAGED>), dim3((unsigned)((rows + 1024 / D - 1) / (1024 / D))), dim3(256), 0, stream, p);
    else if (rows <= 2048) hipLaunchKernelGGL((seq_attn_fold_kernel<D, FMT, PAGED, 4>), dim3((unsigned)rows), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((seq_attn_fold_kernel<D, FMT, PAGED, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, p);
    IGGT_CHECK_LAUNCH();
    return 0;
}

template <int D>
int launch_rows(const SeqAttnParams& p_in, int fmt, hipStream_t stream) {
    SeqAttnParams p = p_in;
    p.qtiles = (int)(((long)p.max_q * p.G + 15) / 16);
    const long n = (long)p.splits * p.qtiles * p.B * p.Hkv;
    if (n >= (1L << 31)) return -4;
    p.items = (unsigned)n;
    const dim3 grid = seq_grid(n), block(256);
    if (fmt == FMT_F16) {
        if (p.max_q == 1) hipLaunchKernelGGL((seq_attn_rows_kernel<D, FMT_F16, false>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((seq_attn_rows_kernel<D, FMT_F16, true>), grid, block, 0, stream, p);
    } else {
        if (p.max_q == 1) hipLaunchKernelGGL((seq_attn_rows_kernel<D, FMT_BF16, false>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((seq_attn_rows_kernel<D, FMT_BF16, true>), grid, block, 0, stream, p);
    }
    IGGT_CHECK_LAUNCH();
    return 0;
}

// Few rows per (request, key head): the row kernel, a work item for every 16 of them.  Its own work grows with the 16-row tiles, the
// tile kernel's hardly up to 128 rows, but that one reads and converts keys at a lower rate.  Measured, rows / tile kernel, us: 16
// requests of 4 096 tokens, 4 key heads of 128: 32 rows 36 / 33 (29 and a fold of 7), 64 rows 26 / 38 (not split), 128 rows 48 / 51; of 64:
// 21 / 26, 18 / 25, 26 / 30; 32 requests of 2 048, 16 key heads of 64: 32 rows 41 / 53, 64 rows 76 / 53; of 128: 88 / 99, 154 / 92; 2 of
// 16 384, 16 heads of 128: 64 rows 64 / 70, 128 rows 108 / 76.  (Few items, long: 40 000 tokens, 2 heads, 128 rows 19 / 31 and 31 / 51.)
bool few_rows(int B, long max_q, long max_len, int Hkv, int G) {
    const long rows = max_q * G, items = (long)B * Hkv * ((rows + 15) / 16);
    return rows <= 32 || (items <= 1024 && (rows <= 64 || (rows <= 128 && max_len <= 4096)));
}
// Its key ranges are of one length, a multiple of 256 keys, whatever the requests' own lengths, so that requests of different lengths
// fill the chip evenly; the range is as long as leaves about 2 500 work items (three to five rounds of the chip) if all requests had
// max_len tokens, and FOLD_MAX ranges at most (with 128 instead of 64 the fold costs more than the ranges give: 1 x 8 heads of 128, 100 000
// tokens 45 / 37 us, 4 x 2 heads, 60 000 30 / 25).
// Short requests are not split: the fold is a second launch (3.4 us, and as much again of the host's time), a wave's 64 keys are
// 0.5 us (D = 64) or 0.9 us (128).  Measured, split / not: 1 x 16 heads of 64, 1 374 tokens 8.2 / 7.3 us, 2 048 8.1 / 8.8 (in a loop of
// calls 12.9 / 9.5), 4 096 8.6 / 12.8; 4 heads of 128, 1 374 tokens 9.7 / 10.7 (12.8 / 10.8), 2 048 9.7 / 13.3.  Pairs that fill the chip
// gain longer: 16 x 16 heads of 64, 4 096 tokens 25.6 / 21.6.
SeqPlan paged_plan(int B, long max_q, long max_len, int Hkv, int G, int D) {
    if (!few_rows(B, max_q, max_len, Hkv, G)) return iggt_seq_tile_plan(B, max_q, max_len, Hkv, G, D, true);
    const long pairs = (long)B * Hkv * ((max_q * G + 15) / 16), blocks = (max_len + 63) / 64;
    long want = 2560 / pairs;
    if (want > FOLD_MAX) want = FOLD_MAX;
    if (want < 1) want = 1;
    long range = ((blocks + want - 1) / want + 3) / 4 * 4;
    const long single = pairs >= 256 ? 64 : (D == 64 ? 32 : 24);
    if (blocks <= single) range = (blocks + 3) / 4 * 4;
    if (range < 4) range = 4;
    SeqPlan plan = {(int)((blocks + range - 1) / range), false, (int)range};
    if (plan.splits < 1) plan.splits = 1;
    return plan;
}

int page_shift_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

}  // namespace

int iggt_launch_seq_fold(const SeqAttnParams& p, int D, int fmt, bool paged, hipStream_t stream) {
    if (fmt == FMT_F16) {
        if (D == 64) return paged ? launch_fold<64, FMT_F16, true>(p, stream) : launch_fold<64, FMT_F16, false>(p, stream);
        return paged ? launch_fold<128, FMT_F16, true>(p, stream) : launch_fold<128, FMT_F16, false>(p, stream);
    }
    if (D == 64) return paged ? launch_fold<64, FMT_BF16, true>(p, stream) : launch_fold<64, FMT_BF16, false>(p, stream);
    return paged ? launch_fold<128, FMT_BF16, true>(p, stream) : launch_fold<128, FMT_BF16, false>(p, stream);
}

static int paged_attn_h16(int fmt, const void* q, long q_rs, long q_hs, void* o, long o_rs, long o_hs, const void* k_codes,
                          const void* k_scale, const void* v_codes, const void* v_scale, int num_pages, int page,
                          const int* tables, long table_stride, int table_width, const int* lens, const int* cu_q, int B, int Tq,
                          int max_q, int max_len, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                          void* stream) {
    const int shift = page_shift_of(page);
    if (B < 0 || Tq < 0 || max_q < 0 || max_len < 0 || num_pages < 0 || table_width < 0 || shift < 0) return -1;
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return -1;
    if ((long)table_width * page >= (1L << 31) - 1024 || (cu_q == nullptr && max_q > 1) || (long)Tq * Hq >= (1L << 31)) return -1;
    if ((q_rs | q_hs) % 8 || (o_rs | o_hs) % 4 || (uintptr_t)q % 16 || (uintptr_t)o % 8) return -2;
    if (((uintptr_t)k_codes | (uintptr_t)v_codes) % 16) return -2;
    if (!(scale > 0.f && scale <= 1e38f)) return -3;
    if (B == 0 || Tq == 0 || max_q == 0) return 0;
    SeqAttnParams p = {};
    p.q = (const bf16_t*)q; p.o = (bf16_t*)o;
    p.q_rs = q_rs; p.q_hs = q_hs; p.o_rs = o_rs; p.o_hs = o_hs;
    p.k8 = (const uint8_t*)k_codes; p.v8 = (const uint8_t*)v_codes;
    p.k_scale = (const uint8_t*)k_scale; p.v_scale = (const uint8_t*)v_scale;
    p.tables = tables; p.table_stride = table_stride; p.table_width = num_pages > 0 ? table_width : 0; p.lens = lens;
    p.num_pages = num_pages; p.page_shift = shift; p.cu_q = cu_q;
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.Tq = Tq; p.max_q = max_q; p.causal = causal != 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    const SeqPlan plan = paged_plan(B, max_q, max_len, Hkv, p.G, D);
    p.splits = plan.splits;
    p.range_blocks = plan.range_blocks;
    if (p.splits > 1) {
        const long n = (long)p.splits * B * max_q * Hq;
        if (ws == nullptr || ws_len < n * (D + 2) * 4 || (uintptr_t)ws % 16) return -5;
        p.part_o = (float*)ws;
        p.part_ml = p.part_o + n * D;
    }
    const hipStream_t st = (hipStream_t)stream;
    int rc;
    if (few_rows(B, max_q, max_len, Hkv, p.G)) rc = D == 64 ? launch_rows<64>(p, fmt, st) : launch_rows<128>(p, fmt, st);
    else rc = iggt_launch_seq_tiles(p, D, fmt, true, plan.small, st);
    if (rc || p.splits == 1) return rc;
    return iggt_launch_seq_fold(p, D, fmt, true, st);
}

extern "C" {
int iggt_seq_attn_plan(int paged, int B, int max_q, int max_k, int Hq, int Hkv, int D, int* rows, int* ranges) {
    if (B <= 0 || max_q <= 0 || max_k < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return -1;
    const int G = Hq / Hkv;
    const SeqPlan plan = paged ? paged_plan(B, max_q, max_k, Hkv, G, D) : iggt_seq_tile_plan(B, max_q, max_k, Hkv, G, D, false);
    *rows = paged && few_rows(B, max_q, max_k, Hkv, G) ? 16 : (plan.small ? 128 : 256);
    *ranges = plan.splits;
    return 0;
}
long iggt_paged_attn_ws_bytes(int B, int max_q, int max_len, int Hq, int Hkv, int D) {
    if (B <= 0 || max_q <= 0 || max_len < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return 0;
    const SeqPlan plan = paged_plan(B, max_q, max_len, Hkv, Hq / Hkv, D);
    return plan.splits > 1 ? (long)plan.splits * B * max_q * Hq * (D + 2) * 4 : 0;
}
int iggt_paged_attn_bf16(const void* q, long q_rs, long q_hs, void* o, long o_rs, long o_hs, const void* k_codes,
                         const void* k_scale, const void* v_codes, const void* v_scale, int num_pages, int page,
                         const int* tables, long table_stride, int table_width, const int* lens, const int* cu_q, int B, int Tq,
                         int max_q, int max_len, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                         void* stream) {
    return paged_attn_h16(FMT_BF16, q, q_rs, q_hs, o, o_rs, o_hs, k_codes, k_scale, v_codes, v_scale, num_pages, page, tables,
                          table_stride, table_width, lens, cu_q, B, Tq, max_q, max_len, Hq, Hkv, D, scale, causal, ws, ws_len, stream);
}
int iggt_paged_attn_f16(const void* q, long q_rs, long q_hs, void* o, long o_rs, long o_hs, const void* k_codes,
                        const void* k_scale, const void* v_codes, const void* v_scale, int num_pages, int page,
                        const int* tables, long table_stride, int table_width, const int* lens, const int* cu_q, int B, int Tq,
                        int max_q, int max_len, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                        void* stream) {
    return paged_attn_h16(FMT_F16, q, q_rs, q_hs, o, o_rs, o_hs, k_codes, k_scale, v_codes, v_scale, num_pages, page, tables,
                          table_stride, table_width, lens, cu_q, B, Tq, max_q, max_len, Hq, Hkv, D, scale, causal, ws, ws_len, stream);
}
int iggt_seq_call(const long* w) {
    auto in = [w](int i) { return (const void*)w[i]; };
    auto idx = [w](int i) { return (const int*)w[i]; };
    auto out = [w](int i) { return (int*)w[i]; };
    auto num = [w](int i) { return (int)w[i]; };
    auto real = [w](int i) { return (float)__builtin_bit_cast(double, w[i]); };
    switch (w[0]) {
        case IGGT_SEQ_PACKED_ATTN_BF16:
        case IGGT_SEQ_PACKED_ATTN_F16:
            return (w[0] == IGGT_SEQ_PACKED_ATTN_F16 ? iggt_packed_attn_f16 : iggt_packed_attn_bf16)(
                in(1), w[2], w[3], in(4), w[5], w[6], in(7), w[8], w[9], out(10), w[11], w[12], idx(13), idx(14), num(15), num(16), num(17),
                num(18), num(19), num(20), num(21), num(22), real(23), num(24), out(25), w[26], out(27));
        case IGGT_SEQ_PAGED_ATTN_BF16:
        case IGGT_SEQ_PAGED_ATTN_F16:
            return (w[0] == IGGT_SEQ_PAGED_ATTN_F16 ? iggt_paged_attn_f16 : iggt_paged_attn_bf16)(
                in(1), w[2], w[3], out(4), w[5], w[6], in(7), in(8), in(9), in(10), num(11), num(12), idx(13), w[14], num(15), idx(16), idx(17),
                num(18), num(19), num(20), num(21), num(22), num(23), num(24), real(25), num(26), out(27), w[28], out(29));
        case IGGT_SEQ_APPEND_PAGES_BF16:
        case IGGT_SEQ_APPEND_PAGES_F16:
            return (w[0] == IGGT_SEQ_APPEND_PAGES_F16 ? iggt_append_pages_f16 : iggt_append_pages_bf16)(
                in(1), w[2], w[3], in(4), w[5], w[6], idx(7), num(8), out(9), out(10), out(11), out(12), num(13), num(14), num(15), num(16), out(17));
        case IGGT_SEQ_PLAN_PAGES:
            return iggt_plan_pages(out(1), w[2], num(3), num(4), out(5), num(6), idx(7), idx(8), idx(9), num(10), out(11), out(12), out(13),
                                   out(14), num(15), out(16));
    }
    return -1;
}
}
