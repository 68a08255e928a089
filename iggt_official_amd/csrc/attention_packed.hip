// Flash attention over packed sequences of different lengths: causal or not, grouped heads, head dim 64 | 128, 16-bit operands,
// fp32 statistics and accumulators; the same tile kernel serves many query rows over the paged 8-bit cache.
//
// Mathematics (seq_attention.h): online softmax over 64-key tiles.  Swapped product: S^T = K Q^T puts one query row into a lane
// (columns of the 32 x 32 MFMA), so its maximum and sum need one exchange with lane ^ 32, and the numerators P^T leave the
// accumulator already in the layout of the B operand of O^T = V^T P^T: the 8 keys a lane half holds in registers 8u .. 8u + 7 of a
// score block are (r & 3) + 8 (r >> 2) + 4 half, and V^T is fetched for exactly those keys (transposing LDS reads of the row-major
// 16-bit tile; the 8-bit tile is stored transposed already).  The maximum moves only when a row exceeds it by 2^4 (numerators
// stay <= 2^4 above it, or 2^12 with fp16's shift), so the rescale of O and l is rare.
//
// Rounding: scores, maxima, sums and O are fp32; the numerators are rounded to the operand type for the second product (the row sum
// adds them before that rounding), O once on the way out (a mean of values of that type: not saturated, inf and NaN stay).
//
// Values that are not finite: a masked score is replaced, not added to, so NaN in K costs nothing.  V does: 0 * inf = NaN in the
// matrix product.  A tile in which some row sees a key and another does not is therefore scanned (one or two of a row's many); if
// it holds inf or NaN they are added to exactly the rows that see them and the product runs on zeros in their place.
#include "seq_attention.h"
#include "../../include/iggt_hip.h"

using namespace iggt_seq;

namespace {

constexpr float DEFER_THR = 4.0f;

// Order of the work items.  Longest first, so that the last ones to start are short: under a causal mask the last query tiles, else
// the sequences by their number of keys (up to 64 of them: ranked here, one lane each).  Key heads innermost: consecutive workgroups
// go to the XCDs in turn, so one head's tiles share an L2.  Where (sequence, head) pairs are a multiple of 8 but heads are not, an
// XCD would keep one sequence for good: the pairs move on by one every 16th of the tiles.
template <bool PAGED>
IGGT_DEVINL void work_item(const SeqAttnParams& p, int lane, int& split, int& qt, int& b, int& h) {
    int w = blockIdx.x;
    if (p.causal || p.B == 1 || p.B > 64) {
        const int npairs = p.B * p.Hkv;
        int pair = w % npairs;
        w /= npairs;
        split = w % p.splits;
        const int at = w / p.splits;
        qt = p.qtiles - 1 - at;
        pair = (pair + at / ((p.qtiles >> 4) + 1)) % npairs;
        b = pair / p.Hkv;
        h = pair - b * p.Hkv;
    } else {
        h = w % p.Hkv;
        w /= p.Hkv;
        split = w % p.splits;
        w /= p.splits;
        qt = w % p.qtiles;
        const int place = w / p.qtiles;
        const int lk = lane < p.B ? seq_span<PAGED>(p, lane).lk : -1;
        int rank = 0;
        for (int i = 0; i < p.B; ++i) {
            const int other = __builtin_amdgcn_readlane(lk, i);
            rank += (other > lk || (other == lk && i < lane)) ? 1 : 0;
        }
        const unsigned long long mine = __ballot(lane < p.B && rank == place);
        b = (int)__builtin_ctzll(mine);
    }
}

template <int D, int QB, int KVM, int FMT, bool PAGED>
__global__ __launch_bounds__(256, 2) void seq_attn_tile_kernel(const SeqAttnParams p) {
    constexpr int ROWB = D * 2, K_BYTES = 64 * ROWB, TILE = 2 * K_BYTES, BUF = KVM * TILE, NKC = D / 16, NDH = D / 32, BM = 128 * QB;
    constexpr int SLOTS = ROWB / 16;   // 16-byte slots of a K row
    __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int frow = lane & 31, fhalf = lane >> 5;

    int split, qt, b, h;
    work_item<PAGED>(p, lane, split, qt, b, h);
    const SeqSpan sp = seq_span<PAGED>(p, b);
    const long rows = (long)sp.lq * p.G;
    const long row0 = (long)qt * BM;
    if (row0 >= rows) return;
    const int off = sp.lk - sp.lq;
    auto limit_of = [&](long row) {   // keys that row sees
        return p.causal ? max(min(sp.lk, off + (int)(row / p.G) + 1), 0) : sp.lk;
    };
    const int kend = limit_of(min(row0 + BM, rows) - 1);
    const int ktiles = (kend + 63) >> 6;
    const int mtiles = (ktiles + KVM - 1) / KVM;                    // macro tiles of 64 KVM keys: one barrier each
    const int t0 = (int)((long)mtiles * split / p.splits), t1 = (int)((long)mtiles * (split + 1) / p.splits);

    const int wg_first = limit_of(row0);   // keys every row of the tile sees
    const long wrow = row0 + wave * (32 * QB);
    const bool live_wave = wrow < rows;
    const int w_first = live_wave ? limit_of(wrow) : 0;                                   // keys every row of the wave sees
    const int w_last = live_wave ? limit_of(min(wrow + 32 * QB, rows) - 1) : 0;           // keys its last row sees

    bf16x8 qf[QB][NKC];
    int lim[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const long r = min(wrow + qb * 32 + frow, rows - 1);
        const int i = (int)(r / p.G), hq = h * p.G + (int)(r - (long)i * p.G);
        lim[qb] = limit_of(r);
        const bf16_t* src = p.q + (long)(sp.q0 + i) * p.q_rs + (long)hq * p.q_hs + 8 * fhalf;
#pragma unroll
        for (int kc = 0; kc < NKC; ++kc) qf[qb][kc] = *reinterpret_cast<const bf16x8*>(src + 16 * kc);
    }

    // ---- staging.  16-bit: LDS-DMA, 1 KiB per wave and instruction; the row-image swizzles are applied to the source piece, rows
    //      past the end are clamped to the last key (masked; see the file comment for values that are not finite).
    typedef __attribute__((address_space(1))) const void gptr_t;
    typedef __attribute__((address_space(3))) void lptr_t;
    constexpr int RPC = 1024 / ROWB;            // rows of a 1 KiB chunk
    constexpr int CPW = K_BYTES / 1024 / 4;     // chunks per wave
    const bf16_t* kb_ptr = nullptr;
    const bf16_t* vb_ptr = nullptr;
    int drow[CPW], kcol[CPW], vcol[CPW];        // row and swizzled byte column of the lane's piece in each of its chunks
    uint32_t koffs[CPW], voffs[CPW];            // their byte offsets within a tile (host: a tile spans less than 2^32)
    if constexpr (!PAGED) {
        kb_ptr = p.k + (long)sp.k0 * p.k_rs + (long)h * p.k_hs;
        vb_ptr = p.v + (long)sp.k0 * p.v_rs + (long)h * p.v_hs;
#pragma unroll
        for (int i = 0; i < CPW; ++i) {
            const int r = (wave * CPW + i) * RPC + lane / SLOTS, pos = lane % SLOTS;
            drow[i] = r;
            kcol[i] = (D == 64 ? pos ^ ((r >> 1) & 7) : pos ^ (r & 15)) * 16;
            vcol[i] = (D == 64 ? (((pos >> 1) ^ (r & 2)) << 1) | (pos & 1) : (((pos >> 1) ^ ((r & 3) << 1)) << 1) | (pos & 1)) * 16;
            koffs[i] = (uint32_t)r * (uint32_t)(2 * p.k_rs) + kcol[i];
            voffs[i] = (uint32_t)r * (uint32_t)(2 * p.v_rs) + vcol[i];
        }
    }
    auto dma = [&](int mt, int buf) {
#pragma unroll
        for (int sub = 0; sub < KVM; ++sub) {
            const int t = mt * KVM + sub;
            if (KVM > 1 && t >= ktiles) break;
            char* sK = smem + buf * BUF + sub * TILE;
            char* sV = sK + K_BYTES;
            const char* kt = reinterpret_cast<const char*>(kb_ptr + (long)t * 64 * p.k_rs);
            const char* vt = reinterpret_cast<const char*>(vb_ptr + (long)t * 64 * p.v_rs);
            const int left = sp.lk - 1 - t * 64;
            if (left < 63) {
#pragma unroll
                for (int i = 0; i < CPW; ++i) {
                    const uint32_t r = min(drow[i], left);
                    __builtin_amdgcn_global_load_lds((gptr_t*)(kt + (r * (uint32_t)(2 * p.k_rs) + kcol[i])), (lptr_t*)(sK + (wave * CPW + i) * 1024), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((gptr_t*)(vt + (r * (uint32_t)(2 * p.v_rs) + vcol[i])), (lptr_t*)(sV + (wave * CPW + i) * 1024), 16, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < CPW; ++i) {
                    __builtin_amdgcn_global_load_lds((gptr_t*)(kt + koffs[i]), (lptr_t*)(sK + (wave * CPW + i) * 1024), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((gptr_t*)(vt + voffs[i]), (lptr_t*)(sV + (wave * CPW + i) * 1024), 16, 0, 0);
                }
            }
        }
    };
    // 8-bit: codes go through registers (16 bytes each), are converted and written as 16-bit tiles: K rows like above, V transposed
    // [D][64 keys] with the keys of every 16 in the order 0-3, 8-11 | 4-7, 12-15 (what the two lane halves need side by side).
    // fp16 holds half of each value (a code of a scale near fp16's range would round to 2^16): the factor 2 of K goes into the softmax
    // scale, that of V into the epilogue.
    constexpr int PPT = D / 64;   // 16-byte pieces of K (and of V) per thread
    constexpr float HALF = (PAGED && FMT == FMT_F16) ? 0.5f : 1.0f;
    u32x4 k8r[PPT], v8r[PPT];
    uint32_t kbyte[PPT], vbyte[PPT];
    uint32_t have_next = 0xf, have = 0xf;       // which 16-key groups of the tile have a page
    // a wave's piece i lies in one 16-key group: one table entry, loaded a tile ahead (lane l: group l & 3), serves its K and its V
    const int psub = D == 64 ? wave : wave >> 1;
    int pid = 0;
    auto look_up = [&](int t) { pid = page_entry(p, b, t * 64 + (lane & 3) * 16); };
    auto fetch = [&](int t) {
        have_next = (uint32_t)__ballot(page_ok(p, pid)) & 0xfu;
        const int pmask = (1 << p.page_shift) - 1;
#pragma unroll
        for (int i = 0; i < PPT; ++i) {
            const int sub = psub + 2 * i;
            const int id = __builtin_amdgcn_readlane(pid, sub);
            const long head = (long)(page_ok(p, id) ? id : 0) * p.Hkv + h;
            const long at = ((head << p.page_shift) + ((t * 64 + sub * 16) & pmask)) * D;      // of the group's K rows, and of its V
            const int in = D == 64 ? lane * 16 : ((wave & 1) * 64 + lane) * 16;
            k8r[i] = *reinterpret_cast<const u32x4*>(p.k8 + at + in);
            v8r[i] = *reinterpret_cast<const u32x4*>(p.v8 + at + in);
            kbyte[i] = p.k_scale[head];
            vbyte[i] = p.v_scale[head];
        }
    };
    auto stage = [&](int buf) {
        char* sK = smem + buf * BUF;
        char* sV = sK + K_BYTES;
#pragma unroll
        for (int i = 0; i < PPT; ++i) {
            const int sub = psub + 2 * i, in = D == 64 ? lane : (wave & 1) * 64 + lane;     // 16-byte piece of the group
            const int key = sub * 16 + in / (D / 16), piece = in % (D / 16), d = in;
            bf16x8 lo, hi;
            cvt16<FMT>(k8r[i], scale_of(kbyte[i]) * HALF, lo, hi);
            const int sw = D == 64 ? (key >> 1) & 7 : key & 15;
            *reinterpret_cast<bf16x8*>(sK + key * ROWB + ((2 * piece) ^ sw) * 16) = lo;
            *reinterpret_cast<bf16x8*>(sK + key * ROWB + ((2 * piece + 1) ^ sw) * 16) = hi;
            cvt16<FMT>(v8r[i], scale_of(vbyte[i]) * HALF, lo, hi);
            const u32x4 a = __builtin_bit_cast(u32x4, lo), z = __builtin_bit_cast(u32x4, hi);
            const u32x4 x = {a[0], a[1], z[0], z[1]}, y = {a[2], a[3], z[2], z[3]};
            *reinterpret_cast<u32x4*>(sV + swz_off(d, 2 * sub)) = x;
            *reinterpret_cast<u32x4*>(sV + swz_off(d, 2 * sub + 1)) = y;
        }
        have = have_next;
    };

    f32x16 o[QB][NDH];
    float m_run[QB], l_run[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        m_run[qb] = M_INIT;
        l_run[qb] = 0.f;
#pragma unroll
        for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[qb][dh][r] = 0.f;
    }
    const float c = p.scale_log2 * (PAGED && FMT == FMT_F16 ? 2.f : 1.f);

    // lane-dependent LDS offsets
    int koff[NKC], voff[NDH];
#pragma unroll
    for (int kc = 0; kc < NKC; ++kc)
        koff[kc] = frow * ROWB + (D == 64 ? (((2 * kc + fhalf) ^ (frow >> 1)) & 7) << 4 : ((2 * kc + fhalf) ^ (frow & 15)) << 4);
    const int tr_i = lane & 15, tr_g = (lane >> 4) & 1;
    {
        const int vr = 4 * fhalf + (tr_i >> 2);
#pragma unroll
        for (int dh = 0; dh < NDH; ++dh)
            voff[dh] = vr * ROWB + (D == 64 ? ((dh * 2 + tr_g) ^ (vr & 2)) << 5 : ((dh * 2 + tr_g) ^ ((vr & 3) << 1)) << 5) + 8 * (tr_i & 3);
    }
    auto v_frag = [&](const char* sV, int kvh, int cc, int dh) -> bf16x8 {
        if constexpr (PAGED) {
            return *reinterpret_cast<const bf16x8*>(sV + swz_off(dh * 32 + frow, 2 * (2 * kvh + cc) + fhalf));
        } else {
            typedef __attribute__((address_space(3))) short4v lds_s4;
            typedef short short8v __attribute__((ext_vector_type(8)));
            const char* base = sV + (kvh * 32 + 16 * cc) * ROWB + voff[dh];
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base));
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + 8 * ROWB));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    auto qk = [&](const char* sK, int qb, f32x16 (&s)[2]) {
        const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int kc = 0; kc < NKC; ++kc) {
                const bf16x8 kf = *reinterpret_cast<const bf16x8*>(sK + kvh * 32 * ROWB + koff[kc]);
                s[kvh] = mfma32h<FMT>(kf, qf[qb][kc], kc == 0 ? zero : s[kvh]);
            }
    };
    auto sees = [&](int t, int qb, int kvh, int r) {
        const int key = kvh * 32 + (r & 3) + 8 * (r >> 2) + 4 * fhalf;
        return t * 64 + key < lim[qb] && (!PAGED || ((have >> (key >> 4)) & 1));
    };
    auto mask = [&](int t, int qb, f32x16 (&s)[2]) {
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!sees(t, qb, kvh, r)) s[kvh][r] = -INFINITY;
    };
    auto update_max = [&](int qb, const f32x16 (&s)[2]) {
        float mx = s[0][0];
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kvh][r]);
        const uint32_t bits = __builtin_bit_cast(uint32_t, mx);
        const auto sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
        mx = fmaxf(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1])) * c;
        if (__any(mx > m_run[qb] + DEFER_THR)) {
            const float m_new = fmaxf(m_run[qb], mx);
            const float alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
            m_run[qb] = m_new;
            l_run[qb] *= alpha;
#pragma unroll
            for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[qb][dh][r] *= alpha;
        }
    };
    auto exp_pack = [&](int qb, f32x16 (&s)[2], bf16x8 (&pf)[2][2]) {
        const float m = m_run[qb] - (FMT == FMT_F16 ? P_SHIFT_F16 : 0.f);
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh) {
            float e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kvh][r], c, -m));
                ls[r & 3] += e[r];
            }
            pf[kvh][0] = pack8f<FMT>(e);
            pf[kvh][1] = pack8f<FMT>(e + 8);
        }
        l_run[qb] += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    };
    auto pv = [&](const char* sV, int qb, const bf16x8 (&pf)[2][2]) {
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                for (int dh = 0; dh < NDH; ++dh) o[qb][dh] = mfma32h<FMT>(v_frag(sV, kvh, cc, dh), pf[kvh][cc], o[qb][dh]);
    };
    // byte of V's element (key, d) in the LDS tile
    auto v_byte = [&](int key, int d) {
        if constexpr (PAGED)
            return swz_off(d, 2 * (key >> 4) + ((key >> 2) & 1)) + 2 * ((key & 3) + ((key >> 3) & 1) * 4);
        else
            return key * ROWB + (D == 64 ? ((d >> 4) ^ (key & 2)) << 5 : ((d >> 4) ^ ((key & 3) << 1)) << 5) + 2 * (d & 15);
    };
    // a tile whose V holds inf or NaN (workgroup-uniform): advance the maxima first, so that no later rescale of this tile meets
    // the infinities; add them to the rows that see them; leave zeros for the matrix product
    auto absorb_nonfinite = [&](char* sK, char* sV, int t) {
        if (t * 64 < w_last) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                f32x16 s[2];
                qk(sK, qb, s);
                mask(t, qb, s);
                update_max(qb, s);
            }
#pragma unroll 1
            for (int key = 0; key < 64; ++key) {
                if (PAGED && !((have >> (key >> 4)) & 1)) continue;
                int fh = fhalf;
                asm volatile("" : "+v"(fh));   // addresses are formed here, not kept in registers across the tile loop
#pragma unroll
                for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = dh * 32 + (r & 3) + 8 * (r >> 2) + 4 * fh;
                        const uint32_t x = *reinterpret_cast<const uint16_t*>(sV + v_byte(key, d));
                        if (nonfinite2<FMT>(x)) {
                            const float f = h2_lo<FMT>(x);
#pragma unroll
                            for (int qb = 0; qb < QB; ++qb)
                                if (t * 64 + key < lim[qb]) o[qb][dh][r] += f;
                        }
                    }
            }
        }
        __syncthreads();
        for (int i = tid * 4; i < K_BYTES; i += 1024) {
            uint32_t w = *reinterpret_cast<const uint32_t*>(sV + i);
            if (nonfinite2<FMT>(w & 0xffffu)) w &= 0xffff0000u;
            if (nonfinite2<FMT>(w & 0xffff0000u)) w &= 0xffffu;
            *reinterpret_cast<uint32_t*>(sV + i) = w;
        }
        __syncthreads();
    };

    // keeps the packed numerators of the first query block where they are formed, beside the second block's score products
    auto pin = [&](bf16x8 (&pf)[2][2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x4 w = __builtin_bit_cast(u32x4, pf[i >> 1][i & 1]);
            asm volatile("" : "+v"(w));
            pf[i >> 1][i & 1] = __builtin_bit_cast(bf16x8, w);
        }
    };

    if (t0 < t1) {
        if constexpr (PAGED) {
            look_up(t0);
            fetch(t0);
            look_up(t0 + 1);
            stage(t0 & 1);
        } else {
            dma(t0, t0 & 1);
        }
        __syncthreads();   // (drains the DMA as well)
        for (int mt = t0; mt < t1; ++mt) {
            if constexpr (PAGED) {
                // (the last tile fetches itself again: a branch here would make every wait one for all loads)
                fetch(min(mt + 1, t1 - 1));
                look_up(mt + 2);
            } else {
                if (mt + 1 < t1) dma(mt + 1, (mt + 1) & 1);
            }
#pragma unroll
            for (int sub = 0; sub < KVM; ++sub) {
                const int t = mt * KVM + sub;
                if (KVM > 1 && t >= ktiles) break;
                char* sK = smem + (mt & 1) * BUF + sub * TILE;
                char* sV = sK + K_BYTES;
                if ((t + 1) * 64 > wg_first || (PAGED && have != 0xf)) {
                    bool bad = false;
                    for (int i = tid * 16; i < K_BYTES; i += 4096) bad = bad || nonfinite8<FMT>(*reinterpret_cast<const bf16x8*>(sV + i));
                    if (__syncthreads_or(bad)) absorb_nonfinite(sK, sV, t);
                }
                if (t * 64 >= w_last) continue;
                const bool edge = (t + 1) * 64 > w_first || (PAGED && have != 0xf);
                f32x16 s0[2], s1[2];
                bf16x8 pf0[2][2], pf1[2][2];
                qk(sK, 0, s0);
                if (edge) mask(t, 0, s0);
                update_max(0, s0);
                if constexpr (QB == 2) qk(sK, 1, s1);
                exp_pack(0, s0, pf0);
                if constexpr (QB == 2) {
                    pin(pf0);
                    if (edge) mask(t, 1, s1);
                    update_max(1, s1);
                }
                pv(sV, 0, pf0);
                if constexpr (QB == 2) {
                    exp_pack(1, s1, pf1);
                    pv(sV, 1, pf1);
                }
            }
            if constexpr (PAGED) {
                if (mt + 1 < t1) stage((mt + 1) & 1);
            }
            __syncthreads();
        }
    }

#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const float l = l_run[qb] + __shfl_xor(l_run[qb], 32, 64);
        const long r = wrow + qb * 32 + frow;
        if (r >= rows) continue;
        const int i = (int)(r / p.G), hq = h * p.G + (int)(r - (long)i * p.G);
        if (p.splits > 1) {
            const long at = (((long)split * p.B + b) * p.max_q + i) * p.Hq + hq;
            if (fhalf == 0) {
                p.part_ml[2 * at] = m_run[qb];
                p.part_ml[2 * at + 1] = l;
            }
            float* dst = p.part_o + at * D + 4 * fhalf;
            if (l != 0.f) {
#pragma unroll
                for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 w = {o[qb][dh][4 * g], o[qb][dh][4 * g + 1], o[qb][dh][4 * g + 2], o[qb][dh][4 * g + 3]};
                        *reinterpret_cast<f32x4*>(dst + dh * 32 + 8 * g) = w;
                    }
            }
        } else {
            const float inv = l == 0.f ? 0.f : (1.0f / HALF) / l;   // no key seen: 0 (O is 0)
            bf16_t* dst = p.o + (long)(sp.q0 + i) * p.o_rs + (long)hq * p.o_hs + 4 * fhalf;
#pragma unroll
            for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    u32x2 w;
                    w[0] = pack_h2<FMT, false>(o[qb][dh][4 * g + 0] * inv, o[qb][dh][4 * g + 1] * inv);
                    w[1] = pack_h2<FMT, false>(o[qb][dh][4 * g + 2] * inv, o[qb][dh][4 * g + 3] * inv);
                    *reinterpret_cast<u32x2*>(dst + dh * 32 + 8 * g) = w;
                }
        }
    }
}

template <int D, int QB, int KVM, int FMT, bool PAGED>
int launch(const SeqAttnParams& p_in, hipStream_t stream) {
    SeqAttnParams p = p_in;
    p.qtiles = (int)(((long)p.max_q * p.G + 128 * QB - 1) / (128 * QB));
    const long n = (long)p.qtiles * p.splits * p.B * p.Hkv;
    if (n >= (1L << 31)) return -4;
    hipLaunchKernelGGL((seq_attn_tile_kernel<D, QB, KVM, FMT, PAGED>), dim3((unsigned)n), dim3(256), 0, stream, p);
    IGGT_CHECK_LAUNCH();
    return 0;
}

template <int FMT, bool PAGED>
int launch_fmt(const SeqAttnParams& p, int D, bool small, hipStream_t stream) {
    if (D == 128) return launch<128, 1, 1, FMT, PAGED>(p, stream);
    constexpr int KVM = PAGED ? 1 : 2;
    return small ? launch<64, 1, KVM, FMT, PAGED>(p, stream) : launch<64, 2, KVM, FMT, PAGED>(p, stream);
}

}  // namespace

int iggt_launch_seq_tiles(const SeqAttnParams& p, int D, int fmt, bool paged, bool small, hipStream_t stream) {
    if (fmt == FMT_F16) return paged ? launch_fmt<FMT_F16, true>(p, D, small, stream) : launch_fmt<FMT_F16, false>(p, D, small, stream);
    return paged ? launch_fmt<FMT_BF16, true>(p, D, small, stream) : launch_fmt<FMT_BF16, false>(p, D, small, stream);
}

SeqPlan iggt_seq_tile_plan(int B, long max_q, long max_k, int Hkv, int G, int D) {
    SeqPlan plan = {};
    const long rows = max_q * G, pairs = (long)B * Hkv, slots = 512;   // two workgroups on each of 256 CUs
    plan.small = D == 64 && (rows <= 128 || pairs * ((rows + 255) / 256) < slots);
    const int bm = (D == 128 || plan.small) ? 128 : 256;
    const long items = pairs * ((rows + bm - 1) / bm);
    long s = 1;
    if (items < slots) {
        s = slots / (items < 1 ? 1 : items);
        const long most = max_k / 512;      // at least eight tiles per range
        if (s > most) s = most;
        if (s > 32) s = 32;
        if (s < 1) s = 1;
    }
    plan.splits = (int)s;
    return plan;
}

static int packed_attn_h16(int fmt, const void* q, long q_rs, long q_hs, const void* k, long k_rs, long k_hs, const void* v,
                           long v_rs, long v_hs, void* o, long o_rs, long o_hs, const int* cu_q, const int* cu_k, int B, int Tq,
                           int Tk, int max_q, int max_k, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                           void* stream) {
    if (B < 0 || Tq < 0 || Tk < 0 || max_q < 0 || max_k < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return -1;
    if (Tk >= 0x7fffffff - 1024) return -1;
    if ((q_rs | q_hs | k_rs | k_hs | v_rs | v_hs) % 8 || (o_rs | o_hs) % 4) return -2;
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || (uintptr_t)o % 8) return -2;
    if (k_rs < 0 || v_rs < 0 || k_rs >= (1L << 24) || v_rs >= (1L << 24)) return -2;   // 64 rows in 32-bit byte offsets
    if (!(scale > 0.f)) return -3;
    if (B == 0 || Tq == 0 || max_q == 0) return 0;
    SeqAttnParams p = {};
    p.q = (const bf16_t*)q; p.k = (const bf16_t*)k; p.v = (const bf16_t*)v; p.o = (bf16_t*)o;
    p.q_rs = q_rs; p.q_hs = q_hs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_rs = v_rs; p.v_hs = v_hs; p.o_rs = o_rs; p.o_hs = o_hs;
    p.cu_q = cu_q; p.cu_k = cu_k;
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.Tq = Tq; p.Tk = Tk; p.max_q = max_q; p.causal = causal != 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    const SeqPlan plan = iggt_seq_tile_plan(B, max_q, max_k, Hkv, p.G, D);
    p.splits = plan.splits;
    if (p.splits > 1) {
        const long n = (long)p.splits * B * max_q * Hq;
        if (ws == nullptr || ws_len < n * (D + 2) * 4 || (uintptr_t)ws % 16) return -5;
        p.part_o = (float*)ws;
        p.part_ml = p.part_o + n * D;
    }
    const int rc = iggt_launch_seq_tiles(p, D, fmt, false, plan.small, (hipStream_t)stream);
    if (rc || p.splits == 1) return rc;
    return iggt_launch_seq_fold(p, D, fmt, false, (hipStream_t)stream);
}

extern "C" {
long iggt_packed_attn_ws_bytes(int B, int max_q, int max_k, int Hq, int Hkv, int D) {
    if (B <= 0 || max_q <= 0 || max_k < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return 0;
    const SeqPlan plan = iggt_seq_tile_plan(B, max_q, max_k, Hkv, Hq / Hkv, D);
    return plan.splits > 1 ? (long)plan.splits * B * max_q * Hq * (D + 2) * 4 : 0;
}
int iggt_packed_attn_bf16(const void* q, long q_rs, long q_hs, const void* k, long k_rs, long k_hs, const void* v, long v_rs,
                          long v_hs, void* o, long o_rs, long o_hs, const int* cu_q, const int* cu_k, int B, int Tq, int Tk,
                          int max_q, int max_k, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                          void* stream) {
    return packed_attn_h16(FMT_BF16, q, q_rs, q_hs, k, k_rs, k_hs, v, v_rs, v_hs, o, o_rs, o_hs, cu_q, cu_k, B, Tq, Tk, max_q, max_k,
                           Hq, Hkv, D, scale, causal, ws, ws_len, stream);
}
int iggt_packed_attn_f16(const void* q, long q_rs, long q_hs, const void* k, long k_rs, long k_hs, const void* v, long v_rs,
                         long v_hs, void* o, long o_rs, long o_hs, const int* cu_q, const int* cu_k, int B, int Tq, int Tk,
                         int max_q, int max_k, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                         void* stream) {
    return packed_attn_h16(FMT_F16, q, q_rs, q_hs, k, k_rs, k_hs, v, v_rs, v_hs, o, o_rs, o_hs, cu_q, cu_k, B, Tq, Tk, max_q, max_k,
                           Hq, Hkv, D, scale, causal, ws, ws_len, stream);
}
}
